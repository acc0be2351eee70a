// K2a / K2b over the 8-bit paged cache (e4m3 codes [num_blocks][num_kv_heads]
// [16][head_dim] and one f32 scale for each (block, head), fp8.cuh).
//
// Decode (one query row per sequence): out = softmax(scale q K^T) V with
// K = ks[block] * Kc, V = vs[block] * Vc.  HBM-bound: every code is read once,
// 2 * ctx * Hkv * D bytes per layer.  Per block a warp computes the transposed
// products with mma.sync, tokens (or the head's D) in the 16 rows of A, the group's
// query heads in the 8 columns, so a group of up to 8 costs half of what
// heads-in-rows would in MMAs, softmax registers and accumulators:
//     S^T[16 tokens][8 heads] = Kc[16][D] x q^T[D][8]
//     O^T[D][8 heads]        += Vc^T[D][16] x W^T[16][8]
// Codes go to f16 in registers (exact), q by a power of two per head.  (An e4m3 mma.sync
// takes the codes as they are only in name: it widens both operands to f16 itself.)
// V scales ride on the softmax weights: with lv = log2 vs,
//     w = exp2(s + lv - m),  m >= max(s + lv),   O = sum w Vc,   l = sum w / vs
// so a weight is bounded by the largest contribution rather than by the largest
// probability, and O / l is the softmax average.  m only moves when a block exceeds it
// by more than 8 (w <= 2^8), so O is rescaled on those blocks alone.
//
// Schedule.  Up to four or eight neighbouring KV heads are a group, a warp each, walking the same
// blocks side by side (their tiles are neighbours in memory).  The blocks of all (sequence,
// group) pairs, laid end to end, are cut into equal runs, one per warp group of a grid that
// fills the GPU once; a warp's cp.async ring runs on across the pairs of its run.  A pair
// cut by a run's end leaves partial results (m, l, O) in the workspace, joined by a second,
// small kernel.  Equal runs end together.  Where every sequence is short (up to 256
// tokens), or there are more than 2,048 of them, a warp takes whole pairs and nothing is
// joined.
//
// Measured (32 query heads on 8, head_dim 128): 256 sequences of 200 to 1,500 tokens 91 us
// (4.9 TB/s; floor 68), 32 of up to 32k 202 us (5.6 TB/s; floor 171), also where the power
// cap lowers the clock.  What bounds it now is the warps' chains of conversion, mma.sync and
// exponentials, three warps per SM sub-partition: the same copies without them take 169 us as
// 16 KB pieces.  256 sequences of 1,000: groups of 4 heads 104 us (floor 80), groups of 16
// 74 (40), head_dim 64 68 (40).  Tried: such pieces by tensor copies from a loading warp 200 us (210 under
// the cap, 97 for the short sequences), 2 KB tensor copies per warp 221, 16 warps of fewer
// registers 213.
//
// Fragments: ldmatrix (plain for K, transposed for V) on 8-bit rows hands each lane four
// neighbouring codes; the k (for V: m) index inside an MMA is a free permutation, chosen
// so that those four codes are what the lane needs.
//
// Prefill (mma.sync, head_dim 64 and groups that the tensor-memory kernel does
// not take): 64-key tiles staged as f16, rows masked causally at absolute
// positions, the same weights w.  Three short prompts of a tiny model take 6.4 us.  A tile is
// staged, converted and multiplied by the same warps one after the other, which bounds it:
// a fresh prompt of 4,000 takes 424 us with 32 heads of 64 on 8 (floor 40), 769 with 28 of
// 128 on 4 (70).
//
// Semantics follow mu_inference/models/layers.py:700-723, as in attention.cu.
#include <math.h>

#include "abi_util.h"
#include "common.cuh"
#include "fp8.cuh"
#include "prefill_fp8.h"

namespace muk {

// Warps per decode CTA, one CTA per SM (registers: 168 or 255 a thread), blocks on their way
// per warp, KV heads side by side at most.  Groups of up to 8 query heads: under the power
// cap, where the chains of a warp take longer, 12 warps in groups of four heads with one block
// ahead take 203 us for 32 sequences of up to 32k and 8 in a group with two ahead 217 (at full
// clock 202 and 196); two ahead of 12 warps were 216, one ahead of 8 warps 222.  Larger groups
// need the registers of 8.
template <int NT>
struct DecodeFp8Shape {
  static constexpr int kWarps = NT == 1 ? 12 : 8;
  static constexpr int kAhead = NT == 1 ? 1 : 2;
  static constexpr int kHeads = NT == 1 ? 4 : 8;
  static constexpr int kStages = 2 + kAhead;  // cp.async ring per warp: two more in work
};
// Blocks of a run, at least: a shorter one costs more in its pair's join than it saves
// (and a pair's partial results stay within kQdMaxParts: the bound of a launch lengthens its
// runs from 24,000 tokens on, whatever the contexts are: 8 sequences of 4,000 take 27 us
// under a bound of 4,368, 35 under 32,768 and 71 under 131,072).
constexpr int kQdMinRun = 12;
constexpr int kQdMaxParts = 127;   // partial results of a pair, at most
constexpr int kQdFlatSeqs = 2048;  // sequences whose block counts a CTA adds up

// Byte offset of 16-byte chunk c of row r in a tile of 8-bit rows of D codes,
// XOR-swizzled so that ldmatrix reads eight rows without a bank conflict.
template <int D>
__device__ __forceinline__ uint32_t swz8(int r, int c) {
  if (D == 128) return (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4));
  return (uint32_t)(r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
}

struct DecodeFp8Args {
  const __nv_bfloat16* q;
  int64_t q_stride;
  __nv_bfloat16* out;
  int64_t out_stride;
  const uint8_t* k_cache;
  const uint8_t* v_cache;
  const float* k_scale;
  const float* v_scale;
  const int32_t* block_tables;
  int bt_stride;
  const int32_t* seq_lens;
  int num_q_heads, num_kv_heads, num_blocks;
  float scale_log2;
  int num_seqs;
  int max_blocks;  // blocks of the longest context the launch is sized for
  int max_parts;   // partial results of a pair; 0: warps take whole pairs
  int min_run;     // blocks of a run, at least (keeps a pair within max_parts)
  int heads;       // neighbouring KV heads whose warps walk the same blocks side by side
  int runs;        // of the grid: groups of `heads` warps
  int* starts;     // [num_seqs + 1] blocks before each sequence, for the join
  float* part_o;   // [sequence][query head][max_parts][D], then (m, l) of each
  float* part_ml;
};

// Blocks of sequence b's context; none where it is empty or longer than the launch.
__device__ __forceinline__ int decode_blocks(const int32_t* seq_lens, int b, int max_blocks) {
  const int ctx = seq_lens[b];
  const int n = ctx <= 0 ? 0 : (ctx - 1) / kKvBlock + 1;
  return n > max_blocks ? 0 : n;
}
// Blocks of a run when `total` are spread.
__device__ __forceinline__ int64_t decode_run(int64_t total, int runs, int min_run) {
  const int64_t r = (total + runs - 1) / runs;
  return r < min_run ? min_run : r;
}

template <int D, int NT>
struct DecodeFp8Smem {
  static constexpr int kTile = kKvBlock * D;            // bytes of one K (or V) block
  static constexpr int kStage = 2 * kTile + 16;         // K, V, two scales (+ pad)
  static constexpr int kRing = DecodeFp8Shape<NT>::kWarps * DecodeFp8Shape<NT>::kStages * kStage;
};

// 2^x, one MUFU op (~2 ulp), far below what the f16 weight keeps.
__device__ __forceinline__ float qd_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// A place in the blocks of all (sequence, head group) pairs, laid end to end: h is a group.
struct DecodePlace {
  int b, h, page, nblk;
};

// NT: 8-head column groups (1: groups of up to 8 query heads, 2: up to 16).
template <int D, int NT>
__global__ void __launch_bounds__(DecodeFp8Shape<NT>::kWarps * 32, 1)
    decode_fp8_kernel(const DecodeFp8Args a) {
  // programmatic dependent launch: let the next kernel launch once every CTA
  // of this one runs, and wait for the previous kernel before touching memory
  grid_dep_launch();
  grid_dep_wait();
  using S = DecodeFp8Smem<D, NT>;
  constexpr int kWarps = DecodeFp8Shape<NT>::kWarps, kAhead = DecodeFp8Shape<NT>::kAhead;
  constexpr int kStages = DecodeFp8Shape<NT>::kStages;
  constexpr int kMT = D / 16;   // k steps of S, and m tiles of O
  extern __shared__ __align__(128) uint8_t smem[];
  int* prefix = reinterpret_cast<int*>(smem + S::kRing);  // [num_seqs + 1] blocks before a sequence

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, tq = lane & 3;
  const int Hkv = a.num_kv_heads, G = a.num_q_heads / Hkv;
  // a run belongs to a group of warps, each with a head of its own
  const int wid = (int)blockIdx.x * (kWarps / a.heads) + warp / a.heads, sub = warp % a.heads;
  const int NG = Hkv / a.heads;  // head groups of a sequence

  // rows of empty sequences are zero; too long ones are latched and left out
  for (int b = blockIdx.x; b < a.num_seqs; b += gridDim.x) {
    const int ctx = a.seq_lens[b];
    if (ctx <= 0) {
      for (int i = threadIdx.x; i < a.num_q_heads * D; i += blockDim.x)
        a.out[(int64_t)b * a.out_stride + i] = f_to_bf16(0.f);
    } else if ((ctx - 1) / kKvBlock + 1 > a.max_blocks) {
      if (threadIdx.x == 0) set_device_error(kDevBadIndex);
    }
  }

  // this warp's run: `left` blocks from `at` on
  DecodePlace at = {0, 0, 0, 0};
  int64_t left = 0;
  const bool flat = a.max_parts > 0;
  if (flat) {
    // prefix sums of the block counts, an equal share of the sequences per thread; the first
    // CTA leaves them for the join
    __shared__ int s_sum[kWarps];
    const int per = (a.num_seqs + kWarps * 32 - 1) / (kWarps * 32);
    const int lo = min((int)threadIdx.x * per, a.num_seqs), hi = min(lo + per, a.num_seqs);
    int sum = 0;
    for (int b = lo; b < hi; ++b) sum += decode_blocks(a.seq_lens, b, a.max_blocks);
    int upto = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    if (lane == 31) s_sum[warp] = upto;
    __syncthreads();
    int before = upto - sum;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) before += w < warp ? s_sum[w] : 0;
    for (int b = lo; b < hi; ++b) {
      prefix[b] = before;
      before += decode_blocks(a.seq_lens, b, a.max_blocks);
    }
    if (hi == a.num_seqs) prefix[hi] = before;
    __syncthreads();
    if (blockIdx.x == 0)
      for (int b = threadIdx.x; b <= a.num_seqs; b += blockDim.x) a.starts[b] = prefix[b];
    const int64_t total = (int64_t)prefix[a.num_seqs] * NG;
    const int64_t run = decode_run(total, a.runs, a.min_run);
    const int64_t first = run * wid;
    left = first < total ? min(run, total - first) : 0;
    if (left > 0) {
      int lo = 0, hi = a.num_seqs;  // the last sequence that starts at or before `first`
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if ((int64_t)prefix[mid] * NG <= first) lo = mid; else hi = mid;
      }
      at.b = lo;
      at.nblk = prefix[lo + 1] - prefix[lo];  // > 0: `first` lies in it
      const int64_t rest = first - (int64_t)prefix[lo] * NG;
      at.h = (int)(rest / at.nblk);
      at.page = (int)(rest % at.nblk);
    }
  }
  auto blocks_of = [&](int b) {
    return flat ? prefix[b + 1] - prefix[b] : decode_blocks(a.seq_lens, b, a.max_blocks);
  };
  const int pairs = a.num_seqs * NG;

  for (int pair = wid; flat ? pair == wid : pair < pairs; pair += a.runs) {
    if (!flat) {  // a whole pair
      at.b = pair / NG;
      at.h = pair % NG;
      at.page = 0;
      at.nblk = blocks_of(at.b);
      left = at.nblk;
    }
    if (left <= 0) continue;

    // ---- loads: chunks of up to 32 blocks of one pair, an id per lane, the next
    // chunk's ids on their way
    const uint32_t wbase = smem_u32(smem) + (uint32_t)(warp * kStages * S::kStage);
    DecodePlace nx = at;       // the next chunk's start
    int64_t nx_left = left;    // blocks from there to the run's end
    int cnt = 0, pos = 0, head = 0, ids = 0, nx_cnt = 0, nx_ids = 0;
    auto fetch = [&]() {       // ids of the chunk at nx
      nx_cnt = (int)min((int64_t)min(32, nx.nblk - nx.page), nx_left);
      nx_ids = lane < nx_cnt ? __ldg(a.block_tables + (int64_t)nx.b * a.bt_stride + nx.page + lane) : 0;
    };
    fetch();
    const uint32_t in_off = swz8<D>(lane / (D / 16), lane % (D / 16));
    int to_issue = (int)left;  // a run, or a pair
    int st_in = 0;
    auto issue = [&]() {       // one block and its group (empty behind the run's end)
      if (to_issue > 0) {
        if (pos == cnt) {
          ids = nx_ids;
          if (ids < 0 || ids >= a.num_blocks) {  // (lanes behind the chunk hold 0)
            set_device_error(kDevBadIndex);
            ids = 0;
          }
          cnt = nx_cnt;
          pos = 0;
          head = nx.h * a.heads + sub;
          nx.page += nx_cnt;
          nx_left -= nx_cnt;
          if (nx.page == nx.nblk && nx_left > 0) {  // on to the next pair
            nx.page = 0;
            if (++nx.h == NG) {
              nx.h = 0;
              do {
                ++nx.b;
                nx.nblk = blocks_of(nx.b);
              } while (nx.nblk == 0);
            }
          }
          if (nx_left > 0) fetch();
        }
        const int id = __shfl_sync(0xffffffffu, ids, pos);
        const int64_t tile = (int64_t)id * Hkv + head;
        const uint8_t* ks = a.k_cache + tile * S::kTile + lane * 16;
        const uint8_t* vs = a.v_cache + tile * S::kTile + lane * 16;
        const uint32_t st = wbase + (uint32_t)(st_in * S::kStage);
        // rows 4 (D = 64: 8) apart: the swizzle of a 128-byte row differs in bit 2 of the chunk
        const uint32_t o0 = st + in_off, o1 = D == 128 ? st + (in_off ^ 64u) : o0;
#pragma unroll
        for (int c = 0; c < S::kTile / 512; ++c) {
          const uint32_t o = (c & 1 ? o1 : o0) + c * 512;
          cp_async_16(o, ks + c * 512);
          cp_async_16(o + S::kTile, vs + c * 512);
        }
        if (lane < 2) cp_async_4(st + 2 * S::kTile + 4 * lane, (lane == 0 ? a.k_scale : a.v_scale) + tile);
        ++pos;
        --to_issue;
        st_in = st_in + 1 == kStages ? 0 : st_in + 1;
      }
      cp_async_commit();
    };
#pragma unroll 1
    for (int i = 0; i < kAhead; ++i) issue();

    // ---- pair by pair
    int st_out = 0;
    // ldmatrix: lanes 8i .. 8i + 7 address the rows of matrix i: tokens 0-7 / 8-15 (i & 1) of
    // chunk k / k + 1 (i >> 1).  The swizzle is an XOR of chunk bits, so chunk k is an XOR too.
    const uint32_t k_off = swz8<D>(((lane >> 3) & 1) * 8 + (lane & 7), lane >> 4);
    while (left > 0) {
      const int page0 = at.page, n = (int)min((int64_t)(at.nblk - at.page), left);
      const int ctx = a.seq_lens[at.b];
      const int h0 = (at.h * a.heads + sub) * G;

      // q as the B operand.  Inside a k step the lane's slots 2tq, 2tq + 1, 2tq + 8, 2tq + 9
      // hold columns 4tq .. 4tq + 3 of the step's 16, as ldmatrix hands out the codes.
      uint32_t qb[NT][kMT][2];
      float qf[NT][2];   // scale_log2 / factor of this lane's result heads 2tq, 2tq + 1
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int hd = nt * 8 + g;
        const __nv_bfloat16* qr =
            a.q + (int64_t)at.b * a.q_stride + (int64_t)(h0 + (hd < G ? hd : 0)) * D + tq * 4;
        uint2 raw[kMT];
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < kMT; ++k) {
          raw[k] = hd < G ? *reinterpret_cast<const uint2*>(qr + k * 16) : make_uint2(0u, 0u);
          // |x| of bf16 pairs as bits of f32
          top = max(top, max(max((raw[k].x << 16) & 0x7fffffffu, raw[k].x & 0x7fff0000u),
                             max((raw[k].y << 16) & 0x7fffffffu, raw[k].y & 0x7fff0000u)));
        }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        float up, down;
        row_factor(top, 14, up, down);
#pragma unroll
        for (int k = 0; k < kMT; ++k) {
          const float2 x = unpack_bf16x2(raw[k].x), y = unpack_bf16x2(raw[k].y);
          qb[nt][k][0] = pack_f16x2(x.x * up, x.y * up);
          qb[nt][k][1] = pack_f16x2(y.x * up, y.y * up);
        }
        qf[nt][0] = __shfl_sync(0xffffffffu, down, (2 * tq) * 4) * a.scale_log2;
        qf[nt][1] = __shfl_sync(0xffffffffu, down, (2 * tq + 1) * 4) * a.scale_log2;
      }

      float m_run[NT][2], l_run[NT][2];
      float o[NT][kMT][4];  // m tile t: rows d = 16 t + 2g (0, 1) and + 1 (2, 3), heads 2tq, 2tq + 1
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        m_run[nt][0] = m_run[nt][1] = -INFINITY;
        l_run[nt][0] = l_run[nt][1] = 0.f;
#pragma unroll
        for (int t = 0; t < kMT; ++t) o[nt][t][0] = o[nt][t][1] = o[nt][t][2] = o[nt][t][3] = 0.f;
      }

      // Two blocks at a time: their chains of loads, products and exponentials overlap, and
      // they share the maximum's shuffles.
      for (int i = 0; i < n; i += 2) {
        const bool two = i + 1 < n;  // else the second is absent: no row of it counts
        issue();
        if (two) issue();
        cp_async_wait<kAhead>();
        __syncwarp();
        uint32_t st[2];
        int rows[2];                 // tokens of the sequence from each block on
        float ks[2], lv[2], iv[2];
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const int slot = st_out + p;
          st[p] = wbase + (uint32_t)((slot >= kStages ? slot - kStages : slot) * S::kStage);
          rows[p] = ctx - (page0 + i + p) * kKvBlock;
          ks[p] = clamp_scale(ld_shared_f32(st[p] + 2 * S::kTile));
          const float vs = clamp_scale(ld_shared_f32(st[p] + 2 * S::kTile + 4));
          asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(lv[p]) : "f"(vs));  // exact for powers of two
          asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(iv[p]) : "f"(vs));
        }
        if (!two) {
          rows[1] = 0;
          lv[1] = 0.f;
          iv[1] = 1.f;
        }
        const bool ragged = rows[0] < kKvBlock || rows[1] < kKvBlock;
        st_out += two ? 2 : 1;
        if (st_out >= kStages) st_out -= kStages;

        // S^T: rows = tokens
        float s[2][NT][4];
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            s[p][nt][0] = s[p][nt][1] = s[p][nt][2] = s[p][nt][3] = 0.f;
#pragma unroll
        for (int k = 0; k < kMT; k += 2)
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            // matrices: (tokens 0-7, chunk k), (tokens 8-15, chunk k), then chunk k + 1
            uint32_t r0, r1, r2, r3, a0, a1, a2, a3;
            ldmatrix_x4(st[p] + (k_off ^ (uint32_t)(k << 4)), r0, r1, r2, r3);
            e4m3x4_to_f16x4(r0, a0, a2);
            e4m3x4_to_f16x4(r1, a1, a3);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma_f16_16816(s[p][nt], a0, a1, a2, a3, qb[nt][k][0], qb[nt][k][1]);
            e4m3x4_to_f16x4(r2, a0, a2);
            e4m3x4_to_f16x4(r3, a1, a3);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma_f16_16816(s[p][nt], a0, a1, a2, a3, qb[nt][k + 1][0], qb[nt][k + 1][1]);
          }
        // weights, per head (column) over the tokens
        uint32_t pb[2][NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            const float f0 = ks[p] * qf[nt][0], f1 = ks[p] * qf[nt][1];
#pragma unroll
            for (int e = 0; e < 4; ++e) s[p][nt][e] = fmaf(s[p][nt][e], e & 1 ? f1 : f0, lv[p]);
          }
          if (ragged) {
#pragma unroll
            for (int p = 0; p < 2; ++p)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (g + (e >> 1) * 8 >= rows[p]) s[p][nt][e] = -INFINITY;
          }
          float mx0 = fmaxf(fmaxf(s[0][nt][0], s[0][nt][2]), fmaxf(s[1][nt][0], s[1][nt][2]));
          float mx1 = fmaxf(fmaxf(s[0][nt][1], s[0][nt][3]), fmaxf(s[1][nt][1], s[1][nt][3]));
#pragma unroll
          for (int sh = 4; sh < 32; sh <<= 1) {
            mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, sh));
            mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, sh));
          }
          const bool up0 = mx0 > m_run[nt][0] + 8.f, up1 = mx1 > m_run[nt][1] + 8.f;  // true at first
          if (__any_sync(0xffffffffu, up0 || up1)) {
            const float c0 = up0 ? qd_exp2(m_run[nt][0] - mx0) : 1.f;
            const float c1 = up1 ? qd_exp2(m_run[nt][1] - mx1) : 1.f;
            if (up0) m_run[nt][0] = mx0;
            if (up1) m_run[nt][1] = mx1;
            l_run[nt][0] *= c0;
            l_run[nt][1] *= c1;
#pragma unroll
            for (int t = 0; t < kMT; ++t) {
              o[nt][t][0] *= c0;
              o[nt][t][1] *= c1;
              o[nt][t][2] *= c0;
              o[nt][t][3] *= c1;
            }
          }
          const float mu0 = m_run[nt][0] == -INFINITY ? 0.f : m_run[nt][0];
          const float mu1 = m_run[nt][1] == -INFINITY ? 0.f : m_run[nt][1];
#pragma unroll
          for (int p = 0; p < 2; ++p) {
#pragma unroll
            for (int e = 0; e < 4; ++e) s[p][nt][e] = qd_exp2(s[p][nt][e] - (e & 1 ? mu1 : mu0));
            l_run[nt][0] = fmaf(s[p][nt][0] + s[p][nt][2], iv[p], l_run[nt][0]);
            l_run[nt][1] = fmaf(s[p][nt][1] + s[p][nt][3], iv[p], l_run[nt][1]);
            // weights <= 2^8 in f16: half a step is 2^-11 of the weight (2^-25 at least)
            pb[p][nt][0] = movmatrix_trans(pack_f16x2(s[p][nt][0], s[p][nt][1]));
            pb[p][nt][1] = movmatrix_trans(pack_f16x2(s[p][nt][2], s[p][nt][3]));
          }
        }
        // O^T += Vc^T W^T
#pragma unroll
        for (int c = 0; c < kMT; c += 2)
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            // matrices: (tokens 0-7, chunk c), (tokens 8-15, chunk c), then chunk c + 1
            uint32_t r[4];
            ldmatrix_x4_trans(st[p] + S::kTile + (k_off ^ (uint32_t)(c << 4)), r[0], r[1], r[2], r[3]);
            if (ragged) {  // rows past the end may hold anything: 0 * NaN is not 0
#pragma unroll
              for (int u = 0; u < 4; ++u) {
                const int t0 = (u & 1) * 8 + 2 * tq;
                r[u] &= (t0 < rows[p] ? 0xffffu : 0u) | (t0 + 1 < rows[p] ? 0xffff0000u : 0u);
              }
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              // a lane holds (token 2tq: d, d + 1), (token 2tq + 1: d, d + 1) with d = 2g
              uint32_t a0, a1, a2, a3;
              e4m3x4_to_f16x4(__byte_perm(r[2 * u], 0, 0x3120), a0, a1);
              e4m3x4_to_f16x4(__byte_perm(r[2 * u + 1], 0, 0x3120), a2, a3);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                mma_f16_16816(o[nt][c + u], a0, a1, a2, a3, pb[p][nt][0], pb[p][nt][1]);
            }
          }
        __syncwarp();
      }

      // ---- the pair's end, or the run's
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          l_run[nt][e] += __shfl_xor_sync(0xffffffffu, l_run[nt][e], 4);
          l_run[nt][e] += __shfl_xor_sync(0xffffffffu, l_run[nt][e], 8);
          l_run[nt][e] += __shfl_xor_sync(0xffffffffu, l_run[nt][e], 16);
        }
      if (n == at.nblk) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int hd = nt * 8 + 2 * tq + e;
            if (hd < G) {
              const float inv = 1.f / l_run[nt][e];
              __nv_bfloat16* dst = a.out + (int64_t)at.b * a.out_stride + (int64_t)(h0 + hd) * D + 2 * g;
#pragma unroll
              for (int t = 0; t < kMT; ++t)
                *reinterpret_cast<uint32_t*>(dst + t * 16) =
                    pack_bf16x2(o[nt][t][e] * inv, o[nt][t][e + 2] * inv);
            }
          }
      } else {
        // this run's number among those that share the pair
        const int64_t total = (int64_t)prefix[a.num_seqs] * NG;
        const int64_t start = (int64_t)prefix[at.b] * NG + (int64_t)at.h * at.nblk;
        const int part = wid - (int)(start / decode_run(total, a.runs, a.min_run));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int hd = nt * 8 + 2 * tq + e;
            if (hd < G && part < a.max_parts) {
              const int64_t row = ((int64_t)at.b * a.num_q_heads + h0 + hd) * a.max_parts + part;
              float* dst = a.part_o + row * D + 2 * g;
#pragma unroll
              for (int t = 0; t < kMT; ++t)
                *reinterpret_cast<float2*>(dst + t * 16) = make_float2(o[nt][t][e], o[nt][t][e + 2]);
              if (g == 0) *reinterpret_cast<float2*>(a.part_ml + row * 2) = make_float2(m_run[nt][e], l_run[nt][e]);
            }
          }
      }
      left -= n;
      at.page = 0;
      if (left > 0) {  // on to the next pair (a run leaves one only at its end)
        if (++at.h == NG) {
          at.h = 0;
          do {
            ++at.b;
            at.nblk = blocks_of(at.b);
          } while (at.nblk == 0);
        }
      }
    }
    cp_async_wait<0>();
  }
}

// Joins the partial results of the pairs that several runs share: a warp per (sequence, KV
// head), eight lanes a query head, in one pass with a running maximum, so that the loads of
// several parts and heads are in flight together.
constexpr int kQdJoinWarps = 4;
template <int D>
__global__ void __launch_bounds__(kQdJoinWarps * 32) decode_fp8_merge_kernel(const DecodeFp8Args a) {
  // programmatic dependent launch: let the next kernel launch once every CTA
  // of this one runs, and wait for the previous kernel before touching memory
  grid_dep_launch();
  grid_dep_wait();
  constexpr int kC = D / 8;  // columns of a lane
  const int item = (int)blockIdx.x * kQdJoinWarps + (int)(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int b = item / a.num_kv_heads, h = item - b * a.num_kv_heads;
  if (b >= a.num_seqs) return;
  const int G = a.num_q_heads / a.num_kv_heads, NG = a.num_kv_heads / a.heads;
  const int from = a.starts[b], nblk = a.starts[b + 1] - from;
  const int64_t run = decode_run((int64_t)a.starts[a.num_seqs] * NG, a.runs, a.min_run);
  if (nblk == 0) return;
  const int64_t start = (int64_t)from * NG + (int64_t)(h / a.heads) * nblk;
  const int parts = min((int)((start + nblk - 1) / run - start / run) + 1, a.max_parts);
  if (parts <= 1) return;
  for (int hd = lane >> 3; hd < G; hd += 4) {
    const int64_t row = ((int64_t)b * a.num_q_heads + h * G + hd) * a.max_parts;
    const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + row;
    const float4* po = reinterpret_cast<const float4*>(a.part_o + row * D) + (lane & 7);
    float M = -INFINITY, L = 0.f, O[kC];
#pragma unroll
    for (int c = 0; c < kC; ++c) O[c] = 0.f;
#pragma unroll 2
    for (int s = 0; s < parts; ++s) {
      const float2 p = ml[s];
      float4 v[kC / 4];  // columns 4 (8 c + lane % 8) ..: eight lanes read 128 bytes
#pragma unroll
      for (int c = 0; c < kC / 4; ++c) v[c] = po[(int64_t)s * (D / 4) + 8 * c];
      const float m = fmaxf(M, p.x), mu = m == -INFINITY ? 0.f : m;
      const float keep = qd_exp2(M - mu), add = qd_exp2(p.x - mu);
      M = m;
      L = fmaf(L, keep, p.y != p.y ? p.y : add * p.y);
#pragma unroll
      for (int c = 0; c < kC / 4; ++c) {
        O[4 * c] = fmaf(add, v[c].x, O[4 * c] * keep);
        O[4 * c + 1] = fmaf(add, v[c].y, O[4 * c + 1] * keep);
        O[4 * c + 2] = fmaf(add, v[c].z, O[4 * c + 2] * keep);
        O[4 * c + 3] = fmaf(add, v[c].w, O[4 * c + 3] * keep);
      }
    }
    const float inv = 1.f / L;
    __nv_bfloat16* dst = a.out + (int64_t)b * a.out_stride + (int64_t)(h * G + hd) * D + (lane & 7) * 4;
#pragma unroll
    for (int c = 0; c < kC / 4; ++c) {
      uint32_t* w = reinterpret_cast<uint32_t*>(dst + 32 * c);
      w[0] = pack_bf16x2(O[4 * c] * inv, O[4 * c + 1] * inv);
      w[1] = pack_bf16x2(O[4 * c + 2] * inv, O[4 * c + 3] * inv);
    }
  }
}

// How a launch is spread: runs of equal length over all pairs (max_parts > 0), or
// whole pairs.
struct DecodeFp8Plan {
  int max_parts, min_run;
};
static DecodeFp8Plan decode_fp8_plan(int max_seq_len, int num_seqs) {
  const int max_blocks = (max_seq_len - 1) / kKvBlock + 1;
  DecodeFp8Plan p = {0, 1};
  if (max_blocks <= 16 || num_seqs > kQdFlatSeqs || (int64_t)num_seqs * max_blocks > INT32_MAX) return p;
  // a pair of max_blocks touches at most max_blocks / min_run + 2 runs
  const int least = (max_blocks + kQdMaxParts - 3) / (kQdMaxParts - 2);
  p.min_run = least > kQdMinRun ? least : kQdMinRun;
  p.max_parts = max_blocks / p.min_run + 2;
  return p;
}

// [num_seqs + 1] ints, padded to 16 bytes, then the partial results.
static size_t decode_fp8_starts(int num_seqs) { return ((size_t)num_seqs + 4) / 4 * 16; }
static size_t decode_fp8_workspace(int num_seqs, int num_q_heads, int head_dim, int max_parts) {
  if (max_parts == 0) return 0;
  return decode_fp8_starts(num_seqs) +
         (size_t)num_seqs * num_q_heads * max_parts * ((size_t)head_dim + 2) * sizeof(float);
}

static int sm_count() {
  static std::atomic<int> count[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  int n = count[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
    count[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

template <int D, int NT>
static int launch_decode_fp8(DecodeFp8Args a, cudaStream_t stream) {
  using Shape = DecodeFp8Shape<NT>;
  constexpr size_t most = DecodeFp8Smem<D, NT>::kRing + (kQdFlatSeqs + 1) * sizeof(int);
  static_assert(most <= 232448 - 64, "decode ring exceeds 227 KB of shared memory");
  const size_t smem = DecodeFp8Smem<D, NT>::kRing + (a.max_parts > 0 ? (a.num_seqs + 1) * sizeof(int) : 0);
  static std::atomic<uint64_t> attr_done{0};
  const cudaError_t ae = smem_attr_once(decode_fp8_kernel<D, NT>, (int)most, attr_done);
  if (ae != cudaSuccess) {
    set_last_error("muk_paged_decode_attn_fp8: cudaFuncSetAttribute: %s", cudaGetErrorString(ae));
    return MUK_ERR_CUDA;
  }
  a.heads = 1;
  while (a.heads < Shape::kHeads && a.num_kv_heads % (2 * a.heads) == 0) a.heads *= 2;
  // a group of warps for each run of the shortest length, or pair, up to one resident grid
  const int64_t pairs = (int64_t)a.num_seqs * (a.num_kv_heads / a.heads);
  const int64_t work = a.max_parts > 0 ? pairs * ((a.max_blocks + a.min_run - 1) / a.min_run) : pairs;
  const int per = Shape::kWarps / a.heads;
  int64_t ctas = (work + per - 1) / per;
  const int64_t fill = sm_count();
  if (ctas > fill) ctas = fill;
  a.runs = (int)ctas * per;
  launch_pdl(decode_fp8_kernel<D, NT>, dim3((unsigned)ctas), dim3(Shape::kWarps * 32), smem, stream, a);
  const int rc = check_launch("muk_paged_decode_attn_fp8");
  if (rc != MUK_OK || a.max_parts == 0) return rc;
  const int64_t items = (int64_t)a.num_seqs * a.num_kv_heads;
  launch_pdl(decode_fp8_merge_kernel<D>, dim3((unsigned)((items + kQdJoinWarps - 1) / kQdJoinWarps)),
             dim3(kQdJoinWarps * 32), 0, stream, a);
  return check_launch("muk_paged_decode_attn_fp8(merge)");
}

// ---------------------------------------------------------------------------
// Prefill on mma.sync: a CTA serves G query heads of one KV head (WR warps of 16
// rows each per head) over 64-key tiles.
// ---------------------------------------------------------------------------
constexpr int kQpKeys = 64;
constexpr int kQpBlocks = kQpKeys / kKvBlock;

// Byte offset of 16-byte chunk c (8 f16) of row r in a staged tile.
template <int D>
__device__ __forceinline__ uint32_t swz16(int r, int c) {
  return (uint32_t)(r * (D * 2) + ((c ^ (r & 7)) << 4));
}

template <int D, int G, int WR>
__global__ void __launch_bounds__(G * WR * 32) prefill_fp8_kernel(const PrefillFp8Args a) {
  // programmatic dependent launch: let the next kernel launch once every CTA
  // of this one runs, and wait for the previous kernel before touching memory
  grid_dep_launch();
  grid_dep_wait();
  constexpr int kThreads = G * WR * 32;
  constexpr int kKS = D / 16, kDT = D / 8;
  constexpr int kRows = 16 * WR;
  constexpr int kTile = kQpKeys * D * 2;            // one staged f16 tile
  constexpr int kUnits = kQpKeys * D / 16;          // 16-code units of a tile
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float s_scale[3][kQpBlocks];           // ks, log2 vs, 1 / vs of the tile's blocks

  const int b = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, tq = lane & 3;
  const int hq = warp / WR, wr = warp % WR;
  const int h = blockIdx.y * G + hq;
  const int q_begin = a.cu_q[b];
  const int q_len = a.cu_q[b + 1] - q_begin;
  const int qt = (int)gridDim.x - 1 - (int)blockIdx.x;  // longest (last) query tiles first
  const int row0 = qt * kRows;
  if (row0 >= q_len) return;
  const int ctx = a.seq_lens[b];
  const int past = ctx - q_len;
  const int kvh = (blockIdx.y * G) / (a.num_q_heads / a.num_kv_heads);
  const int last_q = min(row0 + kRows, q_len) - 1;
  const int n_keys = past + last_q + 1;
  const int nblk = (n_keys - 1) / kKvBlock + 1;
  // uniform: the launch does not cover this sequence
  if (past < 0 || nblk > a.max_blocks || q_begin < 0 || q_len > a.max_q_len ||
      q_begin > a.num_rows - q_len) {
    if (threadIdx.x == 0) set_device_error(kDevBadShape);
    return;
  }
  const int ntiles = (n_keys - 1) / kQpKeys + 1;
  const int32_t* bt = a.block_tables + (int64_t)b * a.bt_stride;
  const uint32_t sk = smem_u32(smem), sv = sk + kTile;

  // q rows g and g + 8 of this warp as A fragments, scaled into f16 per row
  uint32_t qa[kKS][4];
  float qf[2];
  const int qi0 = row0 + wr * 16 + g, qi1 = qi0 + 8;
#pragma unroll
  for (int hr = 0; hr < 2; ++hr) {
    const int qi = hr ? qi1 : qi0;
    const bool live = qi < q_len;
    const __nv_bfloat16* src = a.q + (int64_t)(q_begin + (live ? qi : 0)) * a.q_stride + (int64_t)h * D;
    uint32_t raw[kKS][2], top = 0;
#pragma unroll
    for (int ks = 0; ks < kKS; ++ks)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint32_t v = live ? *reinterpret_cast<const uint32_t*>(src + ks * 16 + u * 8 + tq * 2) : 0u;
        raw[ks][u] = v;
        top = max(top, max((v << 16) & 0x7fffffffu, v & 0x7fff0000u));
      }
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    float up, down;
    row_factor(top, 14, up, down);
    qf[hr] = down * a.scale_log2;
#pragma unroll
    for (int ks = 0; ks < kKS; ++ks)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const float2 x = unpack_bf16x2(raw[ks][u]);
        qa[ks][2 * u + hr] = pack_f16x2(x.x * up, x.y * up);
      }
  }

  float m_row[2] = {-INFINITY, -INFINITY}, l_row[2] = {0.f, 0.f};
  float o[kDT][4];
#pragma unroll
  for (int i = 0; i < kDT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;

  for (int t = 0; t < ntiles; ++t) {
    __syncthreads();  // the previous tile has been read
    if (threadIdx.x < kQpBlocks) {
      const int blk = t * kQpBlocks + threadIdx.x;
      int id = blk < nblk ? __ldg(bt + blk) : 0;
      if (id < 0 || id >= a.num_blocks) id = 0;
      const int64_t at = (int64_t)id * a.num_kv_heads + kvh;
      const float v = blk < nblk ? clamp_scale(a.v_scale[at]) : 1.f;
      s_scale[0][threadIdx.x] = blk < nblk ? clamp_scale(a.k_scale[at]) : 1.f;
      s_scale[1][threadIdx.x] = log2f(v);
      s_scale[2][threadIdx.x] = 1.f / v;
    }
    for (int u = threadIdx.x; u < kUnits; u += kThreads) {
      const int r = u / (D / 16), c = u % (D / 16);
      const int key = t * kQpKeys + r;
      uint4 kv = make_uint4(0u, 0u, 0u, 0u), vv = kv;
      if (key < n_keys) {  // keys behind the last one this CTA sees stay zero
        int id = __ldg(bt + key / kKvBlock);
        if (id < 0 || id >= a.num_blocks) {
          set_device_error(kDevBadIndex);
          id = 0;
        }
        const int64_t off = (((int64_t)id * a.num_kv_heads + kvh) * kKvBlock + (key % kKvBlock)) * D + c * 16;
        kv = *reinterpret_cast<const uint4*>(a.k_cache + off);
        vv = *reinterpret_cast<const uint4*>(a.v_cache + off);
      }
      uint32_t x[8], y[8];
      e4m3x4_to_f16x4(kv.x, x[0], x[1]);
      e4m3x4_to_f16x4(kv.y, x[2], x[3]);
      e4m3x4_to_f16x4(kv.z, x[4], x[5]);
      e4m3x4_to_f16x4(kv.w, x[6], x[7]);
      e4m3x4_to_f16x4(vv.x, y[0], y[1]);
      e4m3x4_to_f16x4(vv.y, y[2], y[3]);
      e4m3x4_to_f16x4(vv.z, y[4], y[5]);
      e4m3x4_to_f16x4(vv.w, y[6], y[7]);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint32_t at = swz16<D>(r, 2 * c + half);
        *reinterpret_cast<uint4*>(smem + at) =
            make_uint4(x[4 * half], x[4 * half + 1], x[4 * half + 2], x[4 * half + 3]);
        *reinterpret_cast<uint4*>(smem + kTile + at) =
            make_uint4(y[4 * half], y[4 * half + 1], y[4 * half + 2], y[4 * half + 3]);
      }
    }
    __syncthreads();

    float s[8][4];
#pragma unroll
    for (int nt = 0; nt < 8; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
    const int mi = lane >> 3, mr = lane & 7;
#pragma unroll
    for (int np = 0; np < 4; ++np) {
      const int row = np * 16 + (mi >= 2 ? 8 : 0) + mr;
#pragma unroll
      for (int ks = 0; ks < kKS; ++ks) {
        uint32_t b0, b1, b2, b3;
        ldmatrix_x4(sk + swz16<D>(row, 2 * ks + (mi & 1)), b0, b1, b2, b3);
        mma_f16_16816(s[2 * np], qa[ks][0], qa[ks][1], qa[ks][2], qa[ks][3], b0, b1);
        mma_f16_16816(s[2 * np + 1], qa[ks][0], qa[ks][1], qa[ks][2], qa[ks][3], b2, b3);
      }
    }
    // scores of block np (16 keys): times ks, plus log2 vs; causal mask
    const int lim0 = past + qi0, lim1 = past + qi1;
#pragma unroll
    for (int nt = 0; nt < 8; ++nt) {
      const float ks = s_scale[0][nt >> 1], lv = s_scale[1][nt >> 1];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = t * kQpKeys + nt * 8 + tq * 2 + (e & 1);
        const bool seen = key <= (e < 2 ? lim0 : lim1) && key < n_keys;
        s[nt][e] = seen ? fmaf(s[nt][e] * ks, qf[e >> 1], lv) : -INFINITY;
      }
    }
    float corr[2];
#pragma unroll
    for (int hr = 0; hr < 2; ++hr) {
      float mx = -INFINITY;
#pragma unroll
      for (int nt = 0; nt < 8; ++nt) mx = fmaxf(mx, fmaxf(s[nt][2 * hr], s[nt][2 * hr + 1]));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float m_new = fmaxf(m_row[hr], mx);
      const float m_use = m_new == -INFINITY ? 0.f : m_new;
      corr[hr] = exp2f(m_row[hr] - m_use);
      m_row[hr] = m_new;
      float sum = 0.f;
#pragma unroll
      for (int nt = 0; nt < 8; ++nt) {
        s[nt][2 * hr] = exp2f(s[nt][2 * hr] - m_use);
        s[nt][2 * hr + 1] = exp2f(s[nt][2 * hr + 1] - m_use);
        // a block that this row does not see must not reach it even as NaN
        if (t * kQpKeys + (nt >> 1) * kKvBlock <= (hr ? lim1 : lim0))
          sum = fmaf(s[nt][2 * hr] + s[nt][2 * hr + 1], s_scale[2][nt >> 1], sum);
      }
      l_row[hr] = l_row[hr] * corr[hr] + sum;
    }
#pragma unroll
    for (int dt = 0; dt < kDT; ++dt) {
      o[dt][0] *= corr[0];
      o[dt][1] *= corr[0];
      o[dt][2] *= corr[1];
      o[dt][3] *= corr[1];
    }
    // weights <= 1 in f16: half a step is 2^-12 of the weight (2^-25 at least)
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      const uint32_t pa0 = pack_f16x2(s[2 * kk][0], s[2 * kk][1]);
      const uint32_t pa1 = pack_f16x2(s[2 * kk][2], s[2 * kk][3]);
      const uint32_t pa2 = pack_f16x2(s[2 * kk + 1][0], s[2 * kk + 1][1]);
      const uint32_t pa3 = pack_f16x2(s[2 * kk + 1][2], s[2 * kk + 1][3]);
      const int row = kk * 16 + ((mi & 1) ? 8 : 0) + mr;
#pragma unroll
      for (int dt = 0; dt < kDT; dt += 2) {
        uint32_t b0, b1, b2, b3;
        ldmatrix_x4_trans(sv + swz16<D>(row, dt + (mi >> 1)), b0, b1, b2, b3);
        mma_f16_16816(o[dt], pa0, pa1, pa2, pa3, b0, b1);
        mma_f16_16816(o[dt + 1], pa0, pa1, pa2, pa3, b2, b3);
      }
    }
  }

#pragma unroll
  for (int hr = 0; hr < 2; ++hr) {
    l_row[hr] += __shfl_xor_sync(0xffffffffu, l_row[hr], 1);
    l_row[hr] += __shfl_xor_sync(0xffffffffu, l_row[hr], 2);
  }
  const float inv0 = 1.f / l_row[0], inv1 = 1.f / l_row[1];
#pragma unroll
  for (int dt = 0; dt < kDT; ++dt) {
    const int c = dt * 8 + tq * 2;
    if (qi0 < q_len)
      *reinterpret_cast<uint32_t*>(a.out + (int64_t)(q_begin + qi0) * a.out_stride + (int64_t)h * D + c) =
          pack_bf16x2(o[dt][0] * inv0, o[dt][1] * inv0);
    if (qi1 < q_len)
      *reinterpret_cast<uint32_t*>(a.out + (int64_t)(q_begin + qi1) * a.out_stride + (int64_t)h * D + c) =
          pack_bf16x2(o[dt][2] * inv1, o[dt][3] * inv1);
  }
}

template <int D, int G, int WR>
static int launch_prefill_fp8(const PrefillFp8Args& a, int num_seqs, int max_q_len,
                              cudaStream_t stream) {
  constexpr size_t smem = (size_t)2 * kQpKeys * D * 2;
  static std::atomic<uint64_t> attr_done{0};
  const cudaError_t ae = smem_attr_once(prefill_fp8_kernel<D, G, WR>, (int)smem, attr_done);
  if (ae != cudaSuccess) {
    set_last_error("muk_paged_prefill_attn_fp8: cudaFuncSetAttribute: %s", cudaGetErrorString(ae));
    return MUK_ERR_CUDA;
  }
  launch_pdl(prefill_fp8_kernel<D, G, WR>,
             dim3((max_q_len + 16 * WR - 1) / (16 * WR), a.num_q_heads / G, num_seqs),
             dim3(G * WR * 32), smem, stream, a);
  return check_launch("muk_paged_prefill_attn_fp8");
}

template <int D>
static int prefill_fp8(const PrefillFp8Args& a, int num_seqs, int max_q_len, cudaStream_t stream) {
  const int gs = a.num_q_heads / a.num_kv_heads;
  if (gs % 4 == 0) return launch_prefill_fp8<D, 4, 1>(a, num_seqs, max_q_len, stream);
  if (gs % 2 == 0) return launch_prefill_fp8<D, 2, 2>(a, num_seqs, max_q_len, stream);
  return launch_prefill_fp8<D, 1, 4>(a, num_seqs, max_q_len, stream);
}

}  // namespace muk

using namespace muk;

extern "C" size_t muk_decode_attn_fp8_workspace_size(int num_seqs, int num_q_heads, int head_dim,
                                                     int max_seq_len, int block_size) {
  if (num_seqs <= 0 || num_q_heads <= 0 || head_dim <= 0 || max_seq_len <= 0 ||
      block_size != kKvBlock)
    return 0;
  // Batches of more than kQdFlatSeqs sequences need none, but a smaller one may follow, and
  // a shorter longest context may have more partial results (its runs may be shorter).
  const int n = num_seqs < kQdFlatSeqs ? num_seqs : kQdFlatSeqs;
  const int most = ((max_seq_len - 1) / kKvBlock + 1) / kQdMinRun + 2;
  const DecodeFp8Plan p = decode_fp8_plan(max_seq_len, 1);
  return decode_fp8_workspace(n, num_q_heads, head_dim,
                              p.max_parts == 0 ? 0 : most < kQdMaxParts ? most : kQdMaxParts);
}

extern "C" int muk_paged_decode_attn_fp8(const void* q, int64_t q_stride, void* out,
                                         int64_t out_stride, const void* k_cache,
                                         const void* v_cache, const float* k_scale,
                                         const float* v_scale, const int32_t* block_tables,
                                         int block_table_stride, const int32_t* seq_lens,
                                         int num_seqs, int num_q_heads, int num_kv_heads,
                                         int head_dim, int block_size, int num_blocks, float scale,
                                         int max_seq_len, void* workspace, size_t workspace_bytes,
                                         void* stream) {
  MUK_REQUIRE(q && out && k_cache && v_cache && k_scale && v_scale && block_tables && seq_lens,
              "muk_paged_decode_attn_fp8: null pointer");
  MUK_REQUIRE(block_size == kKvBlock, "muk_paged_decode_attn_fp8: block_size must be 16, got %d",
              block_size);
  MUK_REQUIRE(num_kv_heads > 0 && num_kv_heads <= 65535 && num_q_heads > 0 &&
                  num_q_heads % num_kv_heads == 0 && num_q_heads / num_kv_heads <= 16,
              "muk_paged_decode_attn_fp8: GQA group %d/%d must divide and be <= 16", num_q_heads,
              num_kv_heads);
  if (head_dim != 64 && head_dim != 128) {
    set_last_error("muk_paged_decode_attn_fp8: head_dim %d not built (64, 128)", head_dim);
    return MUK_ERR_UNSUPPORTED;
  }
  MUK_REQUIRE(q_stride % 4 == 0 && (reinterpret_cast<uintptr_t>(q) & 7u) == 0 &&
                  out_stride % 2 == 0 && (reinterpret_cast<uintptr_t>(out) & 3u) == 0 &&
                  MUK_ALIGNED16(k_cache) && MUK_ALIGNED16(v_cache),
              "muk_paged_decode_attn_fp8: strides/alignment");
  MUK_REQUIRE(num_seqs <= 1 || out_stride >= (int64_t)num_q_heads * head_dim,
              "muk_paged_decode_attn_fp8: rows of out overlap (stride %lld)", (long long)out_stride);
  MUK_REQUIRE(scale > 0.f && scale <= 3.4e38f, "muk_paged_decode_attn_fp8: scale must be positive");
  MUK_REQUIRE(num_blocks > 0 && max_seq_len > 0 &&
                  (int64_t)block_table_stride * kKvBlock >= max_seq_len,
              "muk_paged_decode_attn_fp8: block table narrower than max_seq_len");
  MUK_REQUIRE(num_seqs <= 65535, "muk_paged_decode_attn_fp8: %d sequences in one call", num_seqs);
  if (num_seqs <= 0) return MUK_OK;
  const DecodeFp8Plan p = decode_fp8_plan(max_seq_len, num_seqs);
  DecodeFp8Args a;
  a.q = reinterpret_cast<const __nv_bfloat16*>(q);
  a.q_stride = q_stride;
  a.out = reinterpret_cast<__nv_bfloat16*>(out);
  a.out_stride = out_stride;
  a.k_cache = reinterpret_cast<const uint8_t*>(k_cache);
  a.v_cache = reinterpret_cast<const uint8_t*>(v_cache);
  a.k_scale = k_scale;
  a.v_scale = v_scale;
  a.block_tables = block_tables;
  a.bt_stride = block_table_stride;
  a.seq_lens = seq_lens;
  a.num_q_heads = num_q_heads;
  a.num_kv_heads = num_kv_heads;
  a.num_blocks = num_blocks;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.max_blocks = (max_seq_len - 1) / kKvBlock + 1;
  a.num_seqs = num_seqs;
  a.max_parts = p.max_parts;
  a.min_run = p.min_run;
  a.heads = a.runs = 0;
  a.starts = nullptr;
  a.part_o = a.part_ml = nullptr;
  if (p.max_parts > 0) {
    const size_t rows = (size_t)num_seqs * num_q_heads * p.max_parts;
    const size_t need = decode_fp8_workspace(num_seqs, num_q_heads, head_dim, p.max_parts);
    if (workspace == nullptr || workspace_bytes < need || !MUK_ALIGNED16(workspace)) {
      set_last_error(
          "muk_paged_decode_attn_fp8: workspace needs %zu bytes (16-byte aligned), got %zu", need,
          workspace_bytes);
      return MUK_ERR_WORKSPACE;
    }
    a.starts = reinterpret_cast<int*>(workspace);
    a.part_o = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + decode_fp8_starts(num_seqs));
    a.part_ml = a.part_o + rows * head_dim;
  }
  const bool wide = num_q_heads / num_kv_heads > 8;
  cudaStream_t s = as_stream(stream);
  if (head_dim == 128)
    return wide ? launch_decode_fp8<128, 2>(a, s)
                : launch_decode_fp8<128, 1>(a, s);
  return wide ? launch_decode_fp8<64, 2>(a, s)
              : launch_decode_fp8<64, 1>(a, s);
}

extern "C" int muk_paged_prefill_attn_fp8(const void* q, int64_t q_stride, void* out,
                                          int64_t out_stride, const void* k_cache,
                                          const void* v_cache, const float* k_scale,
                                          const float* v_scale, const int32_t* block_tables,
                                          int block_table_stride, const int32_t* seq_lens,
                                          const int32_t* cu_seqlens_q, int num_seqs, int num_rows,
                                          int max_q_len, int max_seq_len, int num_q_heads,
                                          int num_kv_heads, int head_dim, int block_size,
                                          int num_blocks, float scale, void* stream) {
  MUK_REQUIRE(q && out && k_cache && v_cache && k_scale && v_scale && block_tables && seq_lens &&
                  cu_seqlens_q,
              "muk_paged_prefill_attn_fp8: null pointer");
  MUK_REQUIRE(block_size == kKvBlock, "muk_paged_prefill_attn_fp8: block_size must be 16, got %d",
              block_size);
  MUK_REQUIRE(num_kv_heads > 0 && num_q_heads > 0 && num_q_heads <= 65535 &&
                  num_q_heads % num_kv_heads == 0,
              "muk_paged_prefill_attn_fp8: heads %d/%d", num_q_heads, num_kv_heads);
  if (head_dim != 64 && head_dim != 128) {
    set_last_error("muk_paged_prefill_attn_fp8: head_dim %d not built (64, 128)", head_dim);
    return MUK_ERR_UNSUPPORTED;
  }
  MUK_REQUIRE(q_stride % 8 == 0 && out_stride % 8 == 0 && MUK_ALIGNED16(q) && MUK_ALIGNED16(out) &&
                  MUK_ALIGNED16(k_cache) && MUK_ALIGNED16(v_cache),
              "muk_paged_prefill_attn_fp8: strides/alignment");
  MUK_REQUIRE(num_rows <= 1 || out_stride >= (int64_t)num_q_heads * head_dim,
              "muk_paged_prefill_attn_fp8: rows of out overlap (stride %lld)", (long long)out_stride);
  MUK_REQUIRE(scale > 0.f && scale <= 3.4e38f, "muk_paged_prefill_attn_fp8: scale must be positive");
  MUK_REQUIRE(num_blocks > 0 && max_seq_len > 0 &&
                  (int64_t)block_table_stride * kKvBlock >= max_seq_len,
              "muk_paged_prefill_attn_fp8: block table narrower than max_seq_len");
  MUK_REQUIRE(num_seqs <= 65535, "muk_paged_prefill_attn_fp8: %d sequences in one call", num_seqs);
  MUK_REQUIRE(max_q_len <= 8 * 65535, "muk_paged_prefill_attn_fp8: %d rows of a sequence", max_q_len);
  if (num_seqs <= 0 || max_q_len <= 0) return MUK_OK;
  PrefillFp8Args a;
  a.q = reinterpret_cast<const __nv_bfloat16*>(q);
  a.q_stride = q_stride;
  a.out = reinterpret_cast<__nv_bfloat16*>(out);
  a.out_stride = out_stride;
  a.k_cache = reinterpret_cast<const uint8_t*>(k_cache);
  a.v_cache = reinterpret_cast<const uint8_t*>(v_cache);
  a.k_scale = k_scale;
  a.v_scale = v_scale;
  a.block_tables = block_tables;
  a.bt_stride = block_table_stride;
  a.seq_lens = seq_lens;
  a.cu_q = cu_seqlens_q;
  a.num_rows = num_rows;
  a.max_q_len = max_q_len;
  a.max_blocks = (max_seq_len - 1) / kKvBlock + 1;
  a.num_q_heads = num_q_heads;
  a.num_kv_heads = num_kv_heads;
  a.num_blocks = num_blocks;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.splits = 1;
  cudaStream_t s = as_stream(stream);
  if (prefill_fp8_tc_supported(head_dim, num_q_heads, num_kv_heads))
    return launch_prefill_fp8_tc(a, num_seqs, max_q_len, s);
  return head_dim == 128 ? prefill_fp8<128>(a, num_seqs, max_q_len, s)
                         : prefill_fp8<64>(a, num_seqs, max_q_len, s);
}
