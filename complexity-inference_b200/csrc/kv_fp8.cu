// K1 for the 8-bit cache: per-head QK-norm (optional), rotate-half RoPE and the
// append to paged e4m3 blocks with one power-of-two f32 scale for each (block,
// KV head).
//
// Mathematics.  For the rows R that a call brings into block p, head h:
//   a = max |x| over R,  e = min { e : a <= 448 2^e } in [-60, 60]
//   block new (R holds its row 0):  e stands
//   else, with the block's exponent e0: e = max(e, e0); where it grew, the older
//   rows become e4m3(code * 2^(e0 - e))
//   codes = e4m3(x * 2^-e),  scale = 2^e
// A power of two keeps the older rows' mantissas when a scale grows (only codes
// that fall into e4m3's subnormals round again), and costs nothing: e4m3's
// precision is relative, so a finer scale would only buy part of one bit at the
// bottom of its range.  A block and head with a non-finite value gets the scale
// NaN and stays so until it starts anew; the attention kernels then read it as
// NaN, as they would a bf16 cache holding that value.
//
// Work.  A run = neighbouring batch rows that land in one block (one sequence's
// new tokens: a single row in a decode step, up to 16 in a prefill).  One warp
// owns one (run, K or V head): all its rows stay in registers between the
// maximum and the rounding, so q|k|v is read once.  q rows are rotated by
// further CTAs of the same launch.
//
// The rotation is a*c - b*s with every product rounded (no fused multiply-add)
// and the QK-norm factor is formed in f64: next to a rounding border of e4m3 the
// last bits of f32 decide, and these make the codes independent of the order of
// a sum.  Everything else follows mu_inference/models/layers.py:671-702.
#include <math.h>

#include "abi_util.h"
#include "common.cuh"
#include "fp8.cuh"

namespace muk {

struct KvFp8Args {
  const __nv_bfloat16* qkv;
  int64_t qkv_stride;
  __nv_bfloat16* q_out;
  int64_t q_out_stride;
  const int32_t* positions;
  const int32_t* slots;
  const float* rope_cos;
  const float* rope_sin;
  int max_pos, num_tokens, num_q_heads, num_kv_heads;
  const float* q_norm_w;
  const float* k_norm_w;
  double qk_eps;
  uint8_t* k_cache;
  uint8_t* v_cache;
  float* k_scale;
  float* v_scale;
  int num_blocks;
  int window;      // batch rows per K/V CTA: the runs that start in them are its own
  int kv_ctas;     // leading CTAs: windows x head groups
  int head_groups; // K/V heads are spread over this many CTAs per window
};

constexpr int kAppendThreads = 256;

// 8 + 8 elements of a head: i0 .. i0+7 of the first half and their partners.
__device__ __forceinline__ void unpack16(const uint4& lo, const uint4& hi, float (&x)[16]) {
  const uint32_t l[4] = {lo.x, lo.y, lo.z, lo.w}, h[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const float2 a = unpack_bf16x2(l[u]), b = unpack_bf16x2(h[u]);
    x[2 * u] = a.x;
    x[2 * u + 1] = a.y;
    x[8 + 2 * u] = b.x;
    x[8 + 2 * u + 1] = b.y;
  }
}

// RMSNorm over the head, whose elements lie in D/16 neighbouring lanes.
template <int D>
__device__ __forceinline__ void head_norm(float (&x)[16], const float* w, int i0, double eps) {
  double ss = 0.0;
#pragma unroll
  for (int u = 0; u < 16; ++u) ss += (double)x[u] * (double)x[u];
#pragma unroll
  for (int m = D / 32; m > 0; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
  const float inv = (float)(1.0 / sqrt(ss / (double)D + eps));
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    x[u] = __fmul_rn(w[i0 + u], __fmul_rn(x[u], inv));
    x[8 + u] = __fmul_rn(w[D / 2 + i0 + u], __fmul_rn(x[8 + u], inv));
  }
}

template <int D>
__device__ __forceinline__ void rotate16(float (&x)[16], const float* rope_cos,
                                         const float* rope_sin, int pos, int i0) {
  const float4* cs = reinterpret_cast<const float4*>(rope_cos + (int64_t)pos * (D / 2) + i0);
  const float4* sn = reinterpret_cast<const float4*>(rope_sin + (int64_t)pos * (D / 2) + i0);
  const float4 c0 = __ldg(cs), c1 = __ldg(cs + 1), s0 = __ldg(sn), s1 = __ldg(sn + 1);
  const float c[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
  const float s[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    const float a = x[u], b = x[8 + u];
    x[u] = __fsub_rn(__fmul_rn(a, c[u]), __fmul_rn(b, s[u]));
    x[8 + u] = __fadd_rn(__fmul_rn(b, c[u]), __fmul_rn(a, s[u]));
  }
}

// Codes of a 16-byte group times `ratio` (<= 1), rounded again.
__device__ __forceinline__ uint4 rescale16(uint4 v, float ratio) {
  uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    uint32_t a, b;
    e4m3x4_to_f16x4(w[u], a, b);
    const float2 x = unpack_f16x2(a), y = unpack_f16x2(b);
    w[u] = f32x4_to_e4m3x4(x.x * ratio, x.y * ratio, y.x * ratio, y.y * ratio);
  }
  return v;
}

// One warp: up to 16 rows t .. t+rows-1, all of one block, of K or V head h.
template <int D>
__device__ __forceinline__ void append_rows(const KvFp8Args& a, int t, int rows, int blk, int slot,
                                            bool is_k, int h) {
  constexpr int kLanes = D / 16;           // lanes of a row
  constexpr int kPer = 32 / kLanes;        // rows at a time
  constexpr int kPass = kKvBlock / kPer;
  const int lane = threadIdx.x & 31;
  const int c = lane % kLanes, sub = lane / kLanes, i0 = c * 8;
  // lane i holds row i's place; of rows naming one slot the last one counts
  const int off = slot - blk * kKvBlock;
  const uint32_t same = __match_any_sync(0xffffffffu, lane < rows ? off : 64 + lane);
  bool valid = lane < rows && (31 - __clz(same)) == lane;
  int pos = lane < rows ? a.positions[t + lane] : 0;
  if (is_k && lane < rows && (pos < 0 || pos >= a.max_pos)) {
    set_device_error(kDevBadIndex);
    valid = false;
    pos = 0;
  }
  const uint32_t vmask = __ballot_sync(0xffffffffu, valid);
  const uint32_t omask = __reduce_or_sync(0xffffffffu, valid ? 1u << off : 0u);
  if (vmask == 0) return;

  const __nv_bfloat16* src = a.qkv + (int64_t)t * a.qkv_stride +
                             (int64_t)(a.num_q_heads + (is_k ? h : a.num_kv_heads + h)) * D;
  const int64_t tile = (int64_t)blk * a.num_kv_heads + h;
  uint8_t* dst = (is_k ? a.k_cache : a.v_cache) + tile * (kKvBlock * D);
  float* sc = (is_k ? a.k_scale : a.v_scale) + tile;
  const bool fresh = (omask & 1u) != 0;
  const float old = fresh ? 0.f : *sc;

  uint4 lo[kPass], hi[kPass];
#pragma unroll
  for (int j = 0; j < kPass; ++j) {
    const int r = j * kPer + sub;
    lo[j] = hi[j] = make_uint4(0u, 0u, 0u, 0u);
    if ((vmask >> r) & 1u) {
      const __nv_bfloat16* row = src + (int64_t)r * a.qkv_stride;
      lo[j] = *reinterpret_cast<const uint4*>(row + i0);
      hi[j] = *reinterpret_cast<const uint4*>(row + D / 2 + i0);
    }
  }
  float x[kPass][16];
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < kPass; ++j) {
    if (j * kPer < rows) {  // uniform
      unpack16(lo[j], hi[j], x[j]);
      if (is_k) {
        if (a.k_norm_w != nullptr) head_norm<D>(x[j], a.k_norm_w, i0, a.qk_eps);
        const int p = __shfl_sync(0xffffffffu, pos, j * kPer + sub);
        rotate16<D>(x[j], a.rope_cos, a.rope_sin, p, i0);
      }
#pragma unroll
      for (int u = 0; u < 16; ++u) top = max(top, __float_as_uint(x[j][u]) & 0x7fffffffu);
    }
  }
  // as integers, infinities and NaN come out above every finite value
  top = __reduce_max_sync(0xffffffffu, top);
  const bool bad = top >= 0x7f800000u || old != old;
  int e = bad ? 0 : scale_exponent(top);
  float ratio = 1.f;
  if (!fresh && !bad) {
    // exponent of the smallest power of two that is not below the old scale
    const uint32_t ob = old > 0.f ? __float_as_uint(old) : 0u;
    int eo = (int)(ob >> 23) - 127 + ((ob & 0x7fffffu) != 0 ? 1 : 0);
    eo = min(max(eo, kScaleExpMin), kScaleExpMax);
    e = max(e, eo);
    ratio = old > 0.f ? old * pow2i(-e) : 0.f;
  }
  if (!fresh && !bad && ratio != 1.f) {  // the block's other rows move to the new scale
    constexpr int kUnits = kKvBlock * D / 16 / 32;
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      const int unit = i * 32 + lane, row = unit / (D / 16);
      if (((omask >> row) & 1u) == 0) {
        uint4* p = reinterpret_cast<uint4*>(dst) + unit;
        *p = rescale16(*p, ratio);
      }
    }
  }
  const float inv = pow2i(-e);
#pragma unroll
  for (int j = 0; j < kPass; ++j) {
    const int r = j * kPer + sub;
    const int o = __shfl_sync(0xffffffffu, off, r);
    if ((vmask >> r) & 1u) {
      uint2 a8, b8;
      a8.x = f32x4_to_e4m3x4(x[j][0] * inv, x[j][1] * inv, x[j][2] * inv, x[j][3] * inv);
      a8.y = f32x4_to_e4m3x4(x[j][4] * inv, x[j][5] * inv, x[j][6] * inv, x[j][7] * inv);
      b8.x = f32x4_to_e4m3x4(x[j][8] * inv, x[j][9] * inv, x[j][10] * inv, x[j][11] * inv);
      b8.y = f32x4_to_e4m3x4(x[j][12] * inv, x[j][13] * inv, x[j][14] * inv, x[j][15] * inv);
      if (bad) a8 = b8 = make_uint2(0u, 0u);  // the scale says NaN; no code does
      *reinterpret_cast<uint2*>(dst + o * D + i0) = a8;
      *reinterpret_cast<uint2*>(dst + o * D + D / 2 + i0) = b8;
    }
  }
  if (lane == 0) *sc = bad ? __int_as_float(0x7fffffff) : pow2i(e);
}

template <int D>
__global__ void __launch_bounds__(kAppendThreads) rope_kv_append_fp8_kernel(const KvFp8Args a) {
  // programmatic dependent launch: let the next kernel launch once every CTA
  // of this one runs, and wait for the previous kernel before touching memory
  grid_dep_launch();
  grid_dep_wait();
  constexpr int kLanes = D / 16;
  constexpr int kWarps = kAppendThreads / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int T = a.num_tokens;

  if ((int)blockIdx.x < a.kv_ctas) {
    const int group = (int)blockIdx.x % a.head_groups;
    const int t0 = (int)blockIdx.x / a.head_groups * a.window;
    const int t1 = min(t0 + a.window, T);
    for (int item = group * kWarps + warp; item < 2 * a.num_kv_heads;
         item += a.head_groups * kWarps) {
      const bool is_k = item < a.num_kv_heads;
      const int h = is_k ? item : item - a.num_kv_heads;
      int prev = t0 > 0 ? a.slots[t0 - 1] : -1;
      prev = prev < 0 ? -1 : prev / kKvBlock;
      for (int t = t0; t < t1;) {
        // lanes 0-15 look at the next rows; `n` of them are in row t's block
        const int slot = lane < kKvBlock && t + lane < T ? a.slots[t + lane] : -1;
        const int blk_l = slot < 0 ? -1 : slot / kKvBlock;
        const int blk = __shfl_sync(0xffffffffu, blk_l, 0);
        const uint32_t in = __ballot_sync(0xffffffffu, lane < kKvBlock && blk_l == blk);
        const int n = in == 0xffffu ? kKvBlock : __ffs(~in) - 1;
        // a run belongs to the window that it starts in
        if (blk < 0 || blk == prev) {
          prev = blk;
          t += blk < 0 ? 1 : n;
          continue;
        }
        if (blk >= a.num_blocks) {
          if (lane == 0) set_device_error(kDevBadIndex);
          prev = blk;
          t += n;
          continue;
        }
        append_rows<D>(a, t, n, blk, slot, is_k, h);
        t += n;
        prev = blk;
        // more than 16 neighbouring rows of one block name some slot twice: go
        // on in order, as a later call would
        while (n == kKvBlock && t < T) {
          __syncwarp();
          const int s2 = lane < kKvBlock && t + lane < T ? a.slots[t + lane] : -1;
          const int b2 = s2 < 0 ? -1 : s2 / kKvBlock;
          const uint32_t in2 = __ballot_sync(0xffffffffu, lane < kKvBlock && b2 == blk);
          const int n2 = in2 == 0xffffu ? kKvBlock : __ffs(~in2) - 1;
          if (n2 == 0) break;
          append_rows<D>(a, t, n2, blk, s2, is_k, h);
          t += n2;
          if (n2 < kKvBlock) break;
        }
      }
    }
    return;
  }

  // q rows: thread = 16 elements of a head
  const int t = (int)blockIdx.x - a.kv_ctas;
  int pos = a.positions[t];
  const bool ok = pos >= 0 && pos < a.max_pos;
  if (!ok) {
    if (threadIdx.x == 0) set_device_error(kDevBadIndex);
    pos = 0;
  }
  const int items = a.num_q_heads * kLanes;
  for (int base = 0; base < items; base += kAppendThreads) {  // uniform: the norm shuffles
    const int item = base + threadIdx.x;
    const bool live = item < items;
    const int h = live ? item / kLanes : 0, i0 = (item % kLanes) * 8;
    const __nv_bfloat16* row = a.qkv + (int64_t)t * a.qkv_stride + (int64_t)h * D;
    const uint4 lo = *reinterpret_cast<const uint4*>(row + i0);
    const uint4 hi = *reinterpret_cast<const uint4*>(row + D / 2 + i0);
    float x[16];
    unpack16(lo, hi, x);
    if (a.q_norm_w != nullptr) head_norm<D>(x, a.q_norm_w, i0, a.qk_eps);
    rotate16<D>(x, a.rope_cos, a.rope_sin, pos, i0);
    if (live && ok) {
      __nv_bfloat16* out = a.q_out + (int64_t)t * a.q_out_stride + (int64_t)h * D;
      uint4 l, g;
      l.x = pack_bf16x2(x[0], x[1]);
      l.y = pack_bf16x2(x[2], x[3]);
      l.z = pack_bf16x2(x[4], x[5]);
      l.w = pack_bf16x2(x[6], x[7]);
      g.x = pack_bf16x2(x[8], x[9]);
      g.y = pack_bf16x2(x[10], x[11]);
      g.z = pack_bf16x2(x[12], x[13]);
      g.w = pack_bf16x2(x[14], x[15]);
      *reinterpret_cast<uint4*>(out + i0) = l;
      *reinterpret_cast<uint4*>(out + D / 2 + i0) = g;
    }
  }
}

}  // namespace muk

using namespace muk;

extern "C" int muk_rope_kv_append_fp8(
    const void* qkv, int64_t qkv_stride, void* q_out, int64_t q_out_stride,
    const int32_t* positions, const int32_t* slot_mapping, const float* rope_cos,
    const float* rope_sin, int max_pos, int num_tokens, int num_q_heads, int num_kv_heads,
    int head_dim, const float* q_norm_w, const float* k_norm_w, float qk_eps, void* k_cache,
    void* v_cache, float* k_scale, float* v_scale, int num_blocks, int block_size, void* stream) {
  MUK_REQUIRE(qkv && q_out && positions && slot_mapping && rope_cos && rope_sin && k_cache &&
                  v_cache && k_scale && v_scale,
              "muk_rope_kv_append_fp8: null pointer");
  MUK_REQUIRE(block_size == kKvBlock, "muk_rope_kv_append_fp8: block_size must be 16, got %d",
              block_size);
  MUK_REQUIRE(num_q_heads > 0 && num_kv_heads > 0 && num_q_heads % num_kv_heads == 0,
              "muk_rope_kv_append_fp8: heads %d/%d", num_q_heads, num_kv_heads);
  MUK_REQUIRE(num_blocks > 0 && num_blocks <= INT32_MAX / kKvBlock && max_pos > 0,
              "muk_rope_kv_append_fp8: bad cache (%d blocks, %d positions)", num_blocks, max_pos);
  if (head_dim != 64 && head_dim != 128) {
    set_last_error("muk_rope_kv_append_fp8: head_dim %d not built (64, 128)", head_dim);
    return MUK_ERR_UNSUPPORTED;
  }
  MUK_REQUIRE(qkv_stride >= (int64_t)(num_q_heads + 2 * num_kv_heads) * head_dim &&
                  q_out_stride >= (int64_t)num_q_heads * head_dim && qkv_stride % 8 == 0 &&
                  q_out_stride % 8 == 0,
              "muk_rope_kv_append_fp8: row strides %lld / %lld must hold the heads and be "
              "multiples of 8",
              (long long)qkv_stride, (long long)q_out_stride);
  MUK_REQUIRE(MUK_ALIGNED16(qkv) && MUK_ALIGNED16(q_out) && MUK_ALIGNED16(k_cache) &&
                  MUK_ALIGNED16(v_cache) && MUK_ALIGNED16(rope_cos) && MUK_ALIGNED16(rope_sin),
              "muk_rope_kv_append_fp8: buffers must be 16-byte aligned");
  if (num_tokens <= 0) return MUK_OK;
  KvFp8Args a;
  a.qkv = reinterpret_cast<const __nv_bfloat16*>(qkv);
  a.qkv_stride = qkv_stride;
  a.q_out = reinterpret_cast<__nv_bfloat16*>(q_out);
  a.q_out_stride = q_out_stride;
  a.positions = positions;
  a.slots = slot_mapping;
  a.rope_cos = rope_cos;
  a.rope_sin = rope_sin;
  a.max_pos = max_pos;
  a.num_tokens = num_tokens;
  a.num_q_heads = num_q_heads;
  a.num_kv_heads = num_kv_heads;
  a.q_norm_w = q_norm_w;
  a.k_norm_w = k_norm_w;
  a.qk_eps = (double)qk_eps;
  a.k_cache = reinterpret_cast<uint8_t*>(k_cache);
  a.v_cache = reinterpret_cast<uint8_t*>(v_cache);
  a.k_scale = k_scale;
  a.v_scale = v_scale;
  a.num_blocks = num_blocks;
  // One row per K/V CTA while the step is small (each row of a decode step is a
  // run of its own); 16-row windows for large steps, whose rows are mostly one
  // block's and would leave 15 of 16 single-row CTAs with nothing to do.
  a.window = num_tokens > 1024 ? kKvBlock : 1;
  a.head_groups = (2 * num_kv_heads + kAppendThreads / 32 - 1) / (kAppendThreads / 32);
  const int64_t kv = (int64_t)((num_tokens + a.window - 1) / a.window) * a.head_groups;
  MUK_REQUIRE(kv + num_tokens <= INT32_MAX, "muk_rope_kv_append_fp8: %d tokens", num_tokens);
  a.kv_ctas = (int)kv;
  const dim3 grid((unsigned)(kv + num_tokens));
  launch_pdl(head_dim == 128 ? rope_kv_append_fp8_kernel<128> : rope_kv_append_fp8_kernel<64>, grid,
             dim3(kAppendThreads), 0, as_stream(stream), a);
  return check_launch("muk_rope_kv_append_fp8");
}
