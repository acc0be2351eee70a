// K2a / K2b over the 8-bit paged cache (e4m3 codes [num_blocks][num_kv_heads]
// [16][head_dim] and one f32 scale for each (block, head), fp8.cuh).
//
// Decode (one query row per sequence): out = softmax(scale q K^T) V with
// K = ks[block] * Kc, V = vs[block] * Vc.  HBM-bound: every code is read once,
// 2 * ctx * Hkv * D bytes per layer.  A CTA owns (sequence, KV head, piece of
// the context); its warps stream the piece's blocks through private cp.async
// rings.  Per block a warp computes the transposed products
//     S^T[16 tokens][8 heads]  = Kc[16][D]  x  q^T[D][8]       (A = codes)
//     O^T[D][8 heads]         += vs * (Vc^T[D][16] x P^T[16][8])
// with mma.sync m16n8k16 in f16: the tokens (or the head's D) fill the M rows
// and the group's query heads the 8 columns, so a group of up to 8 costs half of
// what heads-in-rows would (16 rows, most of them empty), in MMAs, in softmax
// registers and in accumulators.  Codes go to f16 in registers (exact).  The
// block's K scale multiplies S after the product and its V scale the partial
// product before it is added, both in f32.
//
// Fragments: ldmatrix (plain for K, transposed for V) on 8-bit rows hands each
// lane four neighbouring codes; the k (for V: m) index inside an MMA is a free
// permutation, chosen so that those four codes are what the lane needs.
//
// Prefill (mma.sync, head_dim 64 and groups that the tensor-memory kernel does
// not take): 64-key tiles staged as f16, rows masked causally at absolute
// positions.  V scales ride on the softmax weights: with lv = log2 vs,
//     w = exp2(s + lv - m),  m >= max(s + lv),   O = sum w Vc,   l = sum w / vs
// so a weight is bounded by the largest contribution rather than by the largest
// probability, and O / l is the softmax average.
//
// Semantics follow mu_inference/models/layers.py:700-723, as in attention.cu.
#include <math.h>

#include "abi_util.h"
#include "common.cuh"
#include "fp8.cuh"
#include "prefill_fp8.h"

namespace muk {

constexpr int kQdWarps = 4;      // warps per decode CTA
constexpr int kQdStages = 3;     // cp.async ring depth per warp (blocks)
constexpr int kQdMaxSplits = 128;

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
  int max_blocks;  // blocks of the longest context the launch is sized for
  int blocks_per_split, max_splits;
  float* part_o;
  float* part_ml;
};

template <int D>
struct DecodeFp8Smem {
  static constexpr int kTile = kKvBlock * D;            // bytes of one K (or V) block
  static constexpr int kStage = 2 * kTile + 16;         // K, V, two scales (+ pad)
  static constexpr int kRing = kQdWarps * kQdStages * kStage;
};

// NT: 8-head column groups (1: groups of up to 8 query heads, 2: up to 16).
template <int D, int NT>
__global__ void __launch_bounds__(kQdWarps * 32) decode_fp8_kernel(const DecodeFp8Args a) {
  // programmatic dependent launch: let the next kernel launch once every CTA
  // of this one runs, and wait for the previous kernel before touching memory
  grid_dep_launch();
  grid_dep_wait();
  using S = DecodeFp8Smem<D>;
  constexpr int kKS = D / 16;  // k steps of S, and m tiles of O
  extern __shared__ __align__(128) uint8_t smem[];

  const int b = blockIdx.z, kvh = blockIdx.y, split = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, tq = lane & 3;
  const int G = a.num_q_heads / a.num_kv_heads;
  const int h0 = kvh * G;

  const int ctx = a.seq_lens[b];
  if (ctx <= 0) {  // nothing cached: the rows are zero
    if (split == 0)
      for (int i = threadIdx.x; i < G * D; i += blockDim.x)
        a.out[(int64_t)b * a.out_stride + (int64_t)h0 * D + i] = f_to_bf16(0.f);
    return;
  }
  const int nblk = (ctx - 1) / kKvBlock + 1;
  const int blk_begin = split * a.blocks_per_split;
  if (blk_begin >= nblk) return;
  const int blk_end = min(nblk, blk_begin + a.blocks_per_split);
  const int nsplit_b = (nblk - 1) / a.blocks_per_split + 1;
  // A context longer than the launch was sized for would read past its
  // block-table row or write past its split slots: latch the error and skip it.
  if (nblk > a.max_blocks) {
    if (threadIdx.x == 0) set_device_error(kDevBadIndex);
    return;
  }

  const uint32_t wbase = smem_u32(smem) + (uint32_t)(warp * kQdStages * S::kStage);
  const int32_t* bt = a.block_tables + (int64_t)b * a.bt_stride;
  const int my_count = (blk_end - blk_begin - warp + kQdWarps - 1) / kQdWarps;  // may be <= 0

  // Block ids of this warp's next 32 blocks, one per lane.
  int ids = 0;
  auto issue = [&](int i) {
    if ((i & 31) == 0) {
      const int j = blk_begin + warp + (i + lane) * kQdWarps;
      ids = j < blk_end ? __ldg(bt + j) : 0;
      if (ids < 0 || ids >= a.num_blocks) {
        set_device_error(kDevBadIndex);
        ids = 0;
      }
    }
    const int64_t tile = (int64_t)__shfl_sync(0xffffffffu, ids, i & 31) * a.num_kv_heads + kvh;
    const uint8_t* ks = a.k_cache + tile * S::kTile;
    const uint8_t* vs = a.v_cache + tile * S::kTile;
    const uint32_t st = wbase + (uint32_t)((i % kQdStages) * S::kStage);
#pragma unroll
    for (int c = 0; c < S::kTile / 16 / 32; ++c) {
      const int idx = c * 32 + lane;
      const int r = idx / (D / 16), ch = idx % (D / 16);
      cp_async_16(st + swz8<D>(r, ch), ks + idx * 16);
      cp_async_16(st + S::kTile + swz8<D>(r, ch), vs + idx * 16);
    }
    if (lane < 2) cp_async_4(st + 2 * S::kTile + 4 * lane, (lane == 0 ? a.k_scale : a.v_scale) + tile);
  };

#pragma unroll
  for (int s = 0; s < kQdStages - 1; ++s) {
    if (s < my_count) issue(s);
    cp_async_commit();
  }

  // q as the B operand, brought into f16 by a power of two per head.  Element
  // order inside a k step: the lane's k slots 2tq, 2tq+1, 2tq+8, 2tq+9 hold
  // columns 4tq .. 4tq+3 of the step's 16, as ldmatrix hands out the codes.
  uint32_t qb[NT][kKS][2];
  float qf[NT][2];   // scale_log2 / factor of this lane's result heads 2tq, 2tq+1
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int head = nt * 8 + g;
    const __nv_bfloat16* qr = a.q + (int64_t)b * a.q_stride + (int64_t)(h0 + (head < G ? head : 0)) * D;
    uint2 raw[kKS];
    uint32_t top = 0;
#pragma unroll
    for (int ks = 0; ks < kKS; ++ks) {
      raw[ks] = head < G ? *reinterpret_cast<const uint2*>(qr + ks * 16 + tq * 4) : make_uint2(0u, 0u);
      // |x| of bf16 pairs as bits of f32
      top = max(top, max(max((raw[ks].x << 16) & 0x7fffffffu, raw[ks].x & 0x7fff0000u),
                         max((raw[ks].y << 16) & 0x7fffffffu, raw[ks].y & 0x7fff0000u)));
    }
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    float up, down;
    row_factor(top, up, down);
#pragma unroll
    for (int ks = 0; ks < kKS; ++ks) {
      const float2 x = unpack_bf16x2(raw[ks].x), y = unpack_bf16x2(raw[ks].y);
      qb[nt][ks][0] = pack_f16x2(x.x * up, x.y * up);
      qb[nt][ks][1] = pack_f16x2(y.x * up, y.y * up);
    }
    qf[nt][0] = __shfl_sync(0xffffffffu, down, (2 * tq) * 4) * a.scale_log2;
    qf[nt][1] = __shfl_sync(0xffffffffu, down, (2 * tq + 1) * 4) * a.scale_log2;
  }

  float m_run[NT][2], l_run[NT][2];
  float o[NT][kKS][4];  // m tile ks: rows d = 16 ks + 2g (0, 1) and + 1 (2, 3), heads 2tq, 2tq + 1
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    m_run[nt][0] = m_run[nt][1] = -INFINITY;
    l_run[nt][0] = l_run[nt][1] = 0.f;
#pragma unroll
    for (int ks = 0; ks < kKS; ++ks) o[nt][ks][0] = o[nt][ks][1] = o[nt][ks][2] = o[nt][ks][3] = 0.f;
  }

  const int mi = lane >> 3, mr = lane & 7;  // ldmatrix: matrix and row that this lane addresses
  for (int i = 0; i < my_count; ++i) {
    if (i + kQdStages - 1 < my_count) issue(i + kQdStages - 1);
    cp_async_commit();
    cp_async_wait<kQdStages - 1>();
    __syncwarp();
    const uint32_t st = wbase + (uint32_t)((i % kQdStages) * S::kStage);
    const int left = ctx - (blk_begin + warp + i * kQdWarps) * kKvBlock;  // tokens of this block on
    const float ksc = ld_shared_f32(st + 2 * S::kTile), vsc = clamp_scale(ld_shared_f32(st + 2 * S::kTile + 4));

    // S^T: rows = tokens
    float s[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
    for (int c = 0; c < kKS; c += 2) {
      // matrices: (tokens 0-7, chunk c), (tokens 8-15, chunk c), then chunk c + 1
      uint32_t r0, r1, r2, r3;
      ldmatrix_x4(st + swz8<D>((mi & 1) * 8 + mr, c + (mi >> 1)), r0, r1, r2, r3);
      uint32_t a0, a1, a2, a3;
      e4m3x4_to_f16x4(r0, a0, a2);
      e4m3x4_to_f16x4(r1, a1, a3);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) mma_f16_16816(s[nt], a0, a1, a2, a3, qb[nt][c][0], qb[nt][c][1]);
      e4m3x4_to_f16x4(r2, a0, a2);
      e4m3x4_to_f16x4(r3, a1, a3);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        mma_f16_16816(s[nt], a0, a1, a2, a3, qb[nt][c + 1][0], qb[nt][c + 1][1]);
    }
    // online softmax in the log2 domain, per head (column) over the tokens
    uint32_t pb[NT][2];
    const float ks = clamp_scale(ksc);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int e = 0; e < 4; ++e) s[nt][e] *= ks * qf[nt][e & 1];
      if (left < kKvBlock) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (g + (e >> 1) * 8 >= left) s[nt][e] = -INFINITY;
      }
      float corr[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float mx = fmaxf(s[nt][e], s[nt][e + 2]);
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        const float m_new = fmaxf(m_run[nt][e], mx);
        const float m_use = m_new == -INFINITY ? 0.f : m_new;
        corr[e] = exp2f(m_run[nt][e] - m_use);
        m_run[nt][e] = m_new;
        s[nt][e] = exp2f(s[nt][e] - m_use);
        s[nt][e + 2] = exp2f(s[nt][e + 2] - m_use);
        l_run[nt][e] = l_run[nt][e] * corr[e] + (s[nt][e] + s[nt][e + 2]);
      }
#pragma unroll
      for (int t = 0; t < kKS; ++t) {
        o[nt][t][0] *= corr[0];
        o[nt][t][1] *= corr[1];
        o[nt][t][2] *= corr[0];
        o[nt][t][3] *= corr[1];
      }
      // weights <= 1 in f16: half a step is 2^-12 of the weight (2^-25 at least)
      pb[nt][0] = movmatrix_trans(pack_f16x2(s[nt][0], s[nt][1]));
      pb[nt][1] = movmatrix_trans(pack_f16x2(s[nt][2], s[nt][3]));
    }
    // O^T += vs * Vc^T P^T
#pragma unroll
    for (int c = 0; c < kKS; c += 2) {
      // matrices: (tokens 0-7, chunk c), (tokens 8-15, chunk c), then chunk c + 1
      uint32_t r[4];
      ldmatrix_x4_trans(st + S::kTile + swz8<D>((mi & 1) * 8 + mr, c + (mi >> 1)), r[0], r[1], r[2], r[3]);
      if (left < kKvBlock) {  // rows past the end may hold anything: 0 * NaN is not 0
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int t0 = (u & 1) * 8 + 2 * tq;
          r[u] &= (t0 < left ? 0xffffu : 0u) | (t0 + 1 < left ? 0xffff0000u : 0u);
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        // a lane holds (token 2tq: d, d + 1), (token 2tq + 1: d, d + 1) with d = 2g
        const uint32_t x = r[2 * u], y = r[2 * u + 1];
        uint32_t a0, a1, a2, a3;
        e4m3x4_to_f16x4(__byte_perm(x, 0, 0x3120), a0, a1);
        e4m3x4_to_f16x4(__byte_perm(y, 0, 0x3120), a2, a3);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float t[4] = {0.f, 0.f, 0.f, 0.f};
          mma_f16_16816(t, a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[nt][c + u][e] = fmaf(vsc, t[e], o[nt][c + u][e]);
        }
      }
    }
    __syncwarp();
  }
  cp_async_wait<0>();

  // Row sums over the token lanes, then the warps' merge through shared memory
  // (the rings are no longer needed).
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      l_run[nt][e] += __shfl_xor_sync(0xffffffffu, l_run[nt][e], 4);
      l_run[nt][e] += __shfl_xor_sync(0xffffffffu, l_run[nt][e], 8);
      l_run[nt][e] += __shfl_xor_sync(0xffffffffu, l_run[nt][e], 16);
    }
  __syncthreads();
  float* s_o = reinterpret_cast<float*>(smem);        // [warps][8 NT][D]
  float* s_m = s_o + kQdWarps * NT * 8 * D;           // [warps][8 NT]
  float* s_l = s_m + kQdWarps * NT * 8;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int row = warp * NT * 8 + nt * 8 + 2 * tq;
#pragma unroll
    for (int t = 0; t < kKS; ++t) {
      const int d = t * 16 + 2 * g;
      *reinterpret_cast<float2*>(s_o + row * D + d) = make_float2(o[nt][t][0], o[nt][t][2]);
      *reinterpret_cast<float2*>(s_o + (row + 1) * D + d) = make_float2(o[nt][t][1], o[nt][t][3]);
    }
    if (g == 0) {
      s_m[row] = m_run[nt][0];
      s_m[row + 1] = m_run[nt][1];
      s_l[row] = l_run[nt][0];
      s_l[row + 1] = l_run[nt][1];
    }
  }
  __syncthreads();
  for (int idx = threadIdx.x; idx < G * D; idx += blockDim.x) {
    const int row = idx / D, d = idx - row * D;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kQdWarps; ++w) M = fmaxf(M, s_m[w * NT * 8 + row]);
    float L = 0.f, O = 0.f;
#pragma unroll
    for (int w = 0; w < kQdWarps; ++w) {
      const float mw = s_m[w * NT * 8 + row];
      const float sc = mw == -INFINITY ? 0.f : exp2f(mw - M);
      // a warp without blocks has l = 0; one whose scores are NaN passes it on
      const float lw = s_l[w * NT * 8 + row];
      L += lw == 0.f ? 0.f : (lw != lw ? lw : sc * lw);
      O += sc * s_o[(w * NT * 8 + row) * D + d];
    }
    const int h = h0 + row;
    if (nsplit_b == 1) {
      a.out[(int64_t)b * a.out_stride + (int64_t)h * D + d] = f_to_bf16(O / L);
    } else {
      const int64_t pidx = ((int64_t)b * a.num_q_heads + h) * a.max_splits + split;
      a.part_o[pidx * D + d] = O;
      if (d == 0) {
        a.part_ml[pidx * 2] = M;
        a.part_ml[pidx * 2 + 1] = L;
      }
    }
  }
}

// Joins the pieces of every (sequence, head) that has more than one.
template <int D>
__global__ void decode_fp8_merge_kernel(__nv_bfloat16* __restrict__ out, int64_t out_stride,
                                        const int32_t* __restrict__ seq_lens, int num_q_heads,
                                        int max_blocks, int blocks_per_split, int max_splits,
                                        const float* __restrict__ part_o,
                                        const float* __restrict__ part_ml) {
  // programmatic dependent launch: let the next kernel launch once every CTA
  // of this one runs, and wait for the previous kernel before touching memory
  grid_dep_launch();
  grid_dep_wait();
  const int b = blockIdx.y, h = blockIdx.x;
  const int ctx = seq_lens[b];
  if (ctx <= 0) return;
  const int nblk = (ctx - 1) / kKvBlock + 1;
  const int ns = (nblk - 1) / blocks_per_split + 1;
  if (ns <= 1 || nblk > max_blocks) return;  // too long: latched by the decode kernel
  const int64_t base = ((int64_t)b * num_q_heads + h) * max_splits;
  float M = -INFINITY;
  for (int s = 0; s < ns; ++s) M = fmaxf(M, part_ml[(base + s) * 2]);
  for (int d = threadIdx.x; d < D; d += blockDim.x) {
    float L = 0.f, O = 0.f;
    for (int s = 0; s < ns; ++s) {
      const float ms = part_ml[(base + s) * 2], ls = part_ml[(base + s) * 2 + 1];
      const float sc = ms == -INFINITY ? 0.f : exp2f(ms - M);
      L += ls != ls ? ls : sc * ls;
      O += sc * part_o[(base + s) * D + d];
    }
    out[(int64_t)b * out_stride + (int64_t)h * D + d] = f_to_bf16(O / L);
  }
}

// Blocks per piece grow with the batch: large batches fill the GPU with whole
// sequences, small ones need pieces for parallelism.
struct DecodeFp8Split {
  int blocks_per_split, max_splits;
};
static DecodeFp8Split decode_fp8_split(int max_seq_len, int num_seqs) {
  const int max_blocks = (max_seq_len - 1) / kKvBlock + 1;
  int64_t bps = (int64_t)num_seqs * max_blocks / 64;
  if (bps > 64) bps = 64;
  const int least = (max_blocks + kQdMaxSplits - 1) / kQdMaxSplits;
  if (bps < least) bps = least;
  if (bps < 16) bps = 16;
  DecodeFp8Split p;
  p.blocks_per_split = (int)bps;
  p.max_splits = (int)((max_blocks + bps - 1) / bps);
  return p;
}

template <int D, int NT>
static int launch_decode_fp8(DecodeFp8Args a, const DecodeFp8Split& p, int num_seqs,
                             cudaStream_t stream) {
  constexpr size_t merge = (size_t)kQdWarps * NT * 8 * (D + 2) * sizeof(float);
  constexpr size_t ring = DecodeFp8Smem<D>::kRing;
  constexpr size_t smem = ring > merge ? ring : merge;
  static std::atomic<uint64_t> attr_done{0};
  const cudaError_t ae = smem_attr_once(decode_fp8_kernel<D, NT>, (int)smem, attr_done);
  if (ae != cudaSuccess) {
    set_last_error("muk_paged_decode_attn_fp8: cudaFuncSetAttribute: %s", cudaGetErrorString(ae));
    return MUK_ERR_CUDA;
  }
  launch_pdl(decode_fp8_kernel<D, NT>, dim3(p.max_splits, a.num_kv_heads, num_seqs),
             dim3(kQdWarps * 32), smem, stream, a);
  const int rc = check_launch("muk_paged_decode_attn_fp8");
  if (rc != MUK_OK || p.max_splits <= 1) return rc;
  launch_pdl(decode_fp8_merge_kernel<D>, dim3(a.num_q_heads, num_seqs), dim3(D), 0, stream, a.out,
             a.out_stride, a.seq_lens, a.num_q_heads, a.max_blocks, p.blocks_per_split, p.max_splits,
             (const float*)a.part_o, (const float*)a.part_ml);
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
    row_factor(top, up, down);
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
  // Smaller batches take shorter (so more) pieces: size for the largest count of
  // any batch of up to num_seqs sequences.
  size_t rows = 0;
  for (int n = 1; n <= num_seqs; ++n) {
    const DecodeFp8Split p = decode_fp8_split(max_seq_len, n);
    const size_t r = p.max_splits > 1 ? (size_t)n * num_q_heads * p.max_splits : 0;
    if (r > rows) rows = r;
  }
  return rows * ((size_t)head_dim + 2) * sizeof(float);
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
                  MUK_ALIGNED16(k_cache) && MUK_ALIGNED16(v_cache),
              "muk_paged_decode_attn_fp8: strides/alignment");
  MUK_REQUIRE(scale > 0.f && scale <= 3.4e38f, "muk_paged_decode_attn_fp8: scale must be positive");
  MUK_REQUIRE(num_blocks > 0 && max_seq_len > 0 &&
                  (int64_t)block_table_stride * kKvBlock >= max_seq_len,
              "muk_paged_decode_attn_fp8: block table narrower than max_seq_len");
  MUK_REQUIRE(num_seqs <= 65535, "muk_paged_decode_attn_fp8: %d sequences in one call", num_seqs);
  if (num_seqs <= 0) return MUK_OK;
  const DecodeFp8Split p = decode_fp8_split(max_seq_len, num_seqs);
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
  a.blocks_per_split = p.blocks_per_split;
  a.max_splits = p.max_splits;
  a.part_o = a.part_ml = nullptr;
  if (p.max_splits > 1) {
    const size_t rows = (size_t)num_seqs * num_q_heads * p.max_splits;
    const size_t need = rows * ((size_t)head_dim + 2) * sizeof(float);
    if (workspace == nullptr || workspace_bytes < need || !MUK_ALIGNED16(workspace)) {
      set_last_error(
          "muk_paged_decode_attn_fp8: workspace needs %zu bytes (16-byte aligned), got %zu", need,
          workspace_bytes);
      return MUK_ERR_WORKSPACE;
    }
    a.part_o = reinterpret_cast<float*>(workspace);
    a.part_ml = a.part_o + rows * head_dim;
  }
  const bool wide = num_q_heads / num_kv_heads > 8;
  cudaStream_t s = as_stream(stream);
  if (head_dim == 128)
    return wide ? launch_decode_fp8<128, 2>(a, p, num_seqs, s)
                : launch_decode_fp8<128, 1>(a, p, num_seqs, s);
  return wide ? launch_decode_fp8<64, 2>(a, p, num_seqs, s)
              : launch_decode_fp8<64, 1>(a, p, num_seqs, s);
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
  cudaStream_t s = as_stream(stream);
  if (prefill_fp8_tc_supported(head_dim, num_q_heads, num_kv_heads))
    return launch_prefill_fp8_tc(a, num_seqs, max_q_len, s);
  return head_dim == 128 ? prefill_fp8<128>(a, num_seqs, max_q_len, s)
                         : prefill_fp8<64>(a, num_seqs, max_q_len, s);
}
