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
// new tokens: a single row in a decode step, up to 16 in a prefill).  A CTA owns
// the runs that start in a window of rows, for a few K / V heads; a head's 16
// rows are spread over two or four warps, 16 elements a thread, which stay in
// registers between the maximum (exchanged through shared memory) and the
// rounding: q|k|v is read once.  (A whole head in one warp, 64 elements a thread,
// took 242 registers and left one CTA on an SM: 141 us for 8k rows.)  q rows are
// rotated by further CTAs of the same launch.
//
// Bound: HBM by the bytes (q|k|v read, q and codes written): the floor of 8,000 rows of
// 32 + 16 heads of 128 is 29 us.  With QK-norm they take 52 us (3.7 TB/s), bound by
// instructions: 36.7 M, issue slots 69 % busy, f64 sum of squares and products rounded one
// by one; without it 46 us, 21.4 M and 50 %, waiting for loads.  256 decode rows take
// 6.3 us, one 4.3 (an empty launch ~3): a dependent round of loads.
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
  int groups;         // groups of K / V heads that a window CTA works on together
  int groups_per_cta, group_ctas;
  int kv_ctas;        // leading CTAs: windows of rows x group_ctas
  int single_ctas;    // next: rows that are alone in their block; 0: the windows take them too
  int q_tokens;       // the others: q of this many rows each
};

constexpr int kWindow = 16;          // batch rows of a window CTA: the runs that start in them are its own
constexpr int kAppendThreads = 256;
// Resident per SM: 80 registers, enough for the loads ahead of large steps.  (Before those,
// 5 CTAs of 48 registers were faster, 61 us for 8k rows to 80; with them 3 take 52.)
constexpr int kAppendCtas = 3;

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

// RMSNorm over the head, whose elements (bf16 numbers) lie in D/16 neighbouring
// lanes (all lanes of the warp take part, `on` lanes change).  The sum of squares is f64; |x| becomes an f64 by its bits, exponent
// rebiased (a conversion instruction runs at an eighth of the rate), which leaves
// subnormals off by less than 2^-126.  1 / sqrt is f32's estimate and one Newton
// step in f64 (2^-43), rounded to f32.
template <int D>
__device__ __forceinline__ void head_norm(float (&x)[16], const float* w, int i0, double eps, bool on) {
  double ss = 0.0;
#pragma unroll
  for (int u = 0; u < 16; ++u) {
    const double v =
        __hiloint2double((int)(((__float_as_uint(x[u]) & 0x7fffffffu) >> 3) + (896u << 20)), 0);
    ss = fma(v, v, ss);
  }
#pragma unroll
  for (int m = D / 32; m > 0; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
  const double m = ss * (1.0 / D) + eps;
  const double y = (double)rsqrtf((float)m);
  float inv = (float)(y * (1.5 - 0.5 * m * y * y));
  if (!(m > 1e-37 && m < 1e37)) inv = (float)(1.0 / sqrt(m));        // m or y beyond f32: the long way
  if (ss >= 0x1p256) inv = __int_as_float(0x7fffffff);  // infinities and NaN among the elements
  if (on) {
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      x[u] = __fmul_rn(w[i0 + u], __fmul_rn(x[u], inv));
      x[8 + u] = __fmul_rn(w[D / 2 + i0 + u], __fmul_rn(x[8 + u], inv));
    }
  }
}

// cos and sin of 8 neighbouring pairs at a position.
struct Rope8 {
  float4 c0, c1, s0, s1;
};
template <int D>
__device__ __forceinline__ Rope8 load_rope(const KvFp8Args& a, int pos, int i0) {
  const float4* cs = reinterpret_cast<const float4*>(a.rope_cos + (int64_t)pos * (D / 2) + i0);
  const float4* sn = reinterpret_cast<const float4*>(a.rope_sin + (int64_t)pos * (D / 2) + i0);
  return {__ldg(cs), __ldg(cs + 1), __ldg(sn), __ldg(sn + 1)};
}
__device__ __forceinline__ void rotate16(float (&x)[16], const Rope8& r) {
  const float c[8] = {r.c0.x, r.c0.y, r.c0.z, r.c0.w, r.c1.x, r.c1.y, r.c1.z, r.c1.w};
  const float s[8] = {r.s0.x, r.s0.y, r.s0.z, r.s0.w, r.s1.x, r.s1.y, r.s1.z, r.s1.w};
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

// The block's new exponent and what its older codes are multiplied by, from the bits of
// the new rows' largest |x| (top), its old scale and whether it starts anew; `bad`: the
// scale becomes NaN.
struct NewScale {
  int e;
  float ratio;
  bool bad;
};
__device__ __forceinline__ NewScale new_scale(uint32_t top, float old, bool fresh) {
  NewScale n;
  // as integers, infinities and NaN come out above every finite value
  n.bad = top >= 0x7f800000u || (!fresh && old != old);
  n.e = n.bad ? 0 : scale_exponent(top);
  n.ratio = 1.f;
  if (!fresh && !n.bad) {
    // exponent of the smallest power of two that is not below the old scale
    const uint32_t ob = old > 0.f ? __float_as_uint(old) : 0u;
    const int eo = (int)(ob >> 23) - 127 + ((ob & 0x7fffffu) != 0 ? 1 : 0);
    n.e = max(n.e, min(max(eo, kScaleExpMin), kScaleExpMax));
    n.ratio = old > 0.f ? old * pow2i(-n.e) : 0.f;
  }
  return n;
}
__device__ __forceinline__ float scale_value(const NewScale& n) {
  return n.bad ? __int_as_float(0x7fffffff) : pow2i(n.e);
}
// A lane's 8 + 8 elements as codes; the scale says NaN where it has to, no code does.
template <int D>
__device__ __forceinline__ void store_row(uint8_t* row, int i0, const float (&x)[16], const NewScale& n) {
  const float inv = pow2i(-n.e);
  uint2 a8, b8;
  a8.x = f32x4_to_e4m3x4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
  a8.y = f32x4_to_e4m3x4(x[4] * inv, x[5] * inv, x[6] * inv, x[7] * inv);
  b8.x = f32x4_to_e4m3x4(x[8] * inv, x[9] * inv, x[10] * inv, x[11] * inv);
  b8.y = f32x4_to_e4m3x4(x[12] * inv, x[13] * inv, x[14] * inv, x[15] * inv);
  if (n.bad) a8 = b8 = make_uint2(0u, 0u);
  *reinterpret_cast<uint2*>(row + i0) = a8;
  *reinterpret_cast<uint2*>(row + D / 2 + i0) = b8;
}
__device__ __forceinline__ uint32_t top_bits(const float (&x)[16]) {
  uint32_t top = 0;
#pragma unroll
  for (int u = 0; u < 16; ++u) top = max(top, __float_as_uint(x[u]) & 0x7fffffffu);
  return top;
}
__device__ __forceinline__ int block_at(const KvFp8Args& a, int t) {
  const int s = t >= 0 && t < a.num_tokens ? a.slots[t] : -1;
  return s < 0 ? -1 : s / kKvBlock;
}

// A row that is alone in its block in this call (decode): the D / 16 lanes of one
// (row, K or V head) do it by themselves.  All lanes of the warp take part.
template <int D>
__device__ __forceinline__ void append_single(const KvFp8Args& a, int64_t item) {
  constexpr int kLanes = D / 16;
  const int lane = threadIdx.x & 31, c = lane % kLanes, i0 = c * 8;
  const int heads = 2 * a.num_kv_heads;
  const bool in = item < (int64_t)a.num_tokens * heads;
  const int t = in ? (int)(item / heads) : 0, j = in ? (int)(item - (int64_t)t * heads) : 0;
  const bool is_k = j < a.num_kv_heads;
  const int h = is_k ? j : j - a.num_kv_heads;
  const int slot = a.slots[t], blk = slot < 0 ? -1 : slot / kKvBlock;
  bool mine = in && blk >= 0 && block_at(a, t - 1) != blk && block_at(a, t + 1) != blk;
  int pos = a.positions[t];
  if (mine && (blk >= a.num_blocks || (is_k && (pos < 0 || pos >= a.max_pos)))) {
    set_device_error(kDevBadIndex);
    mine = false;
  }
  if (!mine || !is_k) pos = 0;
  const int off = mine ? slot - blk * kKvBlock : 0;
  const int64_t tile = (int64_t)(mine ? blk : 0) * a.num_kv_heads + h;
  uint8_t* dst = (is_k ? a.k_cache : a.v_cache) + tile * (kKvBlock * D);
  float* sc = (is_k ? a.k_scale : a.v_scale) + tile;
  const bool fresh = off == 0;
  const float old = mine ? *sc : 0.f;
  const __nv_bfloat16* row = a.qkv + (int64_t)t * a.qkv_stride + (int64_t)(a.num_q_heads + j) * D;
  const uint4 lo = *reinterpret_cast<const uint4*>(row + i0);
  const uint4 hi = *reinterpret_cast<const uint4*>(row + D / 2 + i0);
  float x[16];
  unpack16(lo, hi, x);
  if (a.k_norm_w != nullptr) head_norm<D>(x, a.k_norm_w, i0, a.qk_eps, is_k);
  if (is_k) rotate16(x, load_rope<D>(a, pos, i0));
  uint32_t top = top_bits(x);
#pragma unroll
  for (int m = kLanes / 2; m > 0; m >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, m));
  const NewScale n = new_scale(top, old, fresh);
  if (!mine) return;
  if (n.ratio != 1.f) {  // the block's other rows move to the new scale
#pragma unroll 4
    for (int r = 0; r < kKvBlock; ++r) {
      uint4* q = reinterpret_cast<uint4*>(dst + r * D) + c;
      if (r != off) *q = rescale16(*q, n.ratio);
    }
  }
  store_row<D>(dst + off * D, i0, x, n);
  if (c == 0) *sc = scale_value(n);
}

// Up to 16 rows, all of block blk, of the K and V heads of groups g0 .. g1 - 1 (kHeads
// neighbouring heads, K first, are a group): lane i < 16 holds batch row tr (-1: none) and
// its slot; of rows naming one slot the last counts.  A warp has kPer rows of a head, its
// lanes 16 elements each.  Every warp of the CTA calls it (one barrier a group); the next
// group's rows are loaded while this one's are worked on.
template <int D>
__device__ __forceinline__ void append_rows(const KvFp8Args& a, int tr, int slot, int blk, int g0,
                                            int g1, uint32_t (*red)[kAppendThreads / 32]) {
  constexpr int kLanes = D / 16;           // lanes of a row
  constexpr int kPer = 32 / kLanes;        // rows of a warp
  constexpr int kWph = kKvBlock / kPer;    // warps of a head
  constexpr int kHeads = kAppendThreads / 32 / kWph;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, wq = warp % kWph;
  const int c = lane % kLanes, i0 = c * 8, r = wq * kPer + lane / kLanes;
  const int off = slot - blk * kKvBlock;
  const uint32_t same = __match_any_sync(0xffffffffu, tr >= 0 ? off : 64 + lane);
  const bool valid = tr >= 0 && (31 - __clz(same)) == lane;
  int pos = tr >= 0 ? a.positions[tr] : 0;
  const bool pos_ok = pos >= 0 && pos < a.max_pos;
  if (tr >= 0 && !pos_ok) {
    set_device_error(kDevBadIndex);
    pos = 0;
  }
  // of K rows those with a position, of V rows all
  const uint32_t vk = __ballot_sync(0xffffffffu, valid && pos_ok), vv = __ballot_sync(0xffffffffu, valid);
  const uint32_t ok = __reduce_or_sync(0xffffffffu, valid && pos_ok ? 1u << off : 0u);
  const uint32_t ov = __reduce_or_sync(0xffffffffu, valid ? 1u << off : 0u);
  const int o = __shfl_sync(0xffffffffu, off, r), p = __shfl_sync(0xffffffffu, pos, r);
  const Rope8 rope = load_rope<D>(a, p, i0);
  const int t = __shfl_sync(0xffffffffu, tr, r);
  const __nv_bfloat16* row = a.qkv + (int64_t)max(t, 0) * a.qkv_stride + (int64_t)a.num_q_heads * D + i0;
  uint4 lo, hi;
  auto load = [&](int g) {
    const int j = g * kHeads + warp / kWph;
    lo = hi = make_uint4(0u, 0u, 0u, 0u);
    if (j < 2 * a.num_kv_heads && t >= 0) {
      lo = *reinterpret_cast<const uint4*>(row + (int64_t)j * D);
      hi = *reinterpret_cast<const uint4*>(row + (int64_t)j * D + D / 2);
    }
  };
  load(g0);
  for (int g = g0; g < g1; ++g) {
    const int j = g * kHeads + warp / kWph;
    const bool live = j < 2 * a.num_kv_heads, is_k = j < a.num_kv_heads;
    const int h = !live ? 0 : (is_k ? j : j - a.num_kv_heads);
    const uint32_t vmask = !live ? 0u : (is_k ? vk : vv), omask = is_k ? ok : ov;
    const bool mine = ((vmask >> r) & 1u) != 0, fresh = (omask & 1u) != 0;
    const int64_t tile = (int64_t)blk * a.num_kv_heads + h;
    uint8_t* dst = (is_k ? a.k_cache : a.v_cache) + tile * (kKvBlock * D);
    float* sc = (is_k ? a.k_scale : a.v_scale) + tile;
    const float old = fresh || !live ? 0.f : *sc;
    float x[16];
    unpack16(lo, hi, x);
    if (g + 1 < g1) load(g + 1);
    if (a.k_norm_w != nullptr) head_norm<D>(x, a.k_norm_w, i0, a.qk_eps, is_k);
    if (is_k) rotate16(x, rope);
    uint32_t top = __reduce_max_sync(0xffffffffu, mine ? top_bits(x) : 0u);
    if (lane == 0) red[g & 1][warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWph; ++w) top = max(top, red[g & 1][warp - wq + w]);
    if (vmask == 0) continue;
    const NewScale n = new_scale(top, old, fresh);
    // the block's other rows move to the new scale; a lane's share is chunk c of row r
    if (n.ratio != 1.f && ((omask >> r) & 1u) == 0) {
      uint4* q = reinterpret_cast<uint4*>(dst + r * D) + c;
      *q = rescale16(*q, n.ratio);
    }
    if (mine) store_row<D>(dst + o * D, i0, x, n);
    // every warp of the head has read the old scale: they met at the barrier
    if (lane == 0 && wq == 0) *sc = scale_value(n);
  }
  __syncthreads();  // red, and what was written here, may be used again
}

template <int D>
__global__ void __launch_bounds__(kAppendThreads, kAppendCtas) rope_kv_append_fp8_kernel(const KvFp8Args a) {
  // programmatic dependent launch: let the next kernel launch once every CTA
  // of this one runs, and wait for the previous kernel before touching memory
  grid_dep_launch();
  grid_dep_wait();
  constexpr int kLanes = D / 16;
  __shared__ uint32_t red[2][kAppendThreads / 32];
  const int lane = threadIdx.x & 31;
  const int T = a.num_tokens;

  if ((int)blockIdx.x < a.kv_ctas) {
    const int g0 = (int)blockIdx.x % a.group_ctas * a.groups_per_cta;
    const int g1 = min(g0 + a.groups_per_cta, a.groups);
    const int t0 = (int)blockIdx.x / a.group_ctas * kWindow;
    const int t1 = min(t0 + kWindow, T);
    int prev = t0 > 0 ? a.slots[t0 - 1] : -1;
    prev = prev < 0 ? -1 : prev / kKvBlock;
    // uniform over the CTA: every warp walks the same rows
    for (int t = t0; t < t1;) {
      // the lanes look at the next rows: n of them are in row t's block
      const int slot = t + lane < T ? a.slots[t + lane] : -1;
      const int blk_l = slot < 0 ? -1 : slot / kKvBlock;
      const int blk = __shfl_sync(0xffffffffu, blk_l, 0);
      const uint32_t in = __ballot_sync(0xffffffffu, blk_l == blk);
      int n = in == 0xffffffffu ? 32 : __ffs(~in) - 1;
      // a run belongs to the window that it starts in
      if (blk < 0 || blk == prev || blk >= a.num_blocks || (n == 1 && a.single_ctas > 0)) {
        if (blk >= a.num_blocks && threadIdx.x == 0) set_device_error(kDevBadIndex);
        prev = blk;
        t += blk < 0 ? 1 : n;
        continue;
      }
      int tr = lane < n ? t + lane : -1, at = slot;
      if (n > kKvBlock) {  // more rows than slots: lane i takes the last row that names slot i
        tr = -1;
        at = blk * kKvBlock + lane;
        n = 0;
        for (int m = 32; m == 32; n += m) {
          const int s2 = t + n + lane < T ? a.slots[t + n + lane] : -1;
          const uint32_t in2 = __ballot_sync(0xffffffffu, s2 >= 0 && s2 / kKvBlock == blk);
          m = in2 == 0xffffffffu ? 32 : __ffs(~in2) - 1;
          for (int i = 0; i < m; ++i)
            if (__shfl_sync(0xffffffffu, s2, i) == at) tr = t + n + i;
        }
      }
      append_rows<D>(a, tr, at, blk, g0, g1, red);
      t += n;
      prev = blk;
    }
    return;
  }

  if ((int)blockIdx.x < a.kv_ctas + a.single_ctas) {
    append_single<D>(a, (int64_t)((int)blockIdx.x - a.kv_ctas) * (kAppendThreads / kLanes) +
                            threadIdx.x / kLanes);
    return;
  }

  // q rows: thread = 16 elements of a head; the next item's are loaded meanwhile
  const int items = a.num_q_heads * kLanes;
  const int tb = ((int)blockIdx.x - a.kv_ctas - a.single_ctas) * a.q_tokens;
  const int total = min(a.q_tokens, T - tb) * items;
  int t = 0, h = 0, pos = 0;
  bool live = false;
  uint4 lo, hi;
  const int i0 = (threadIdx.x % kLanes) * 8;
  auto load = [&](int i) {
    live = i < total;
    t = tb + (live ? i / items : 0);
    h = live ? i % items / kLanes : 0;
    const __nv_bfloat16* row = a.qkv + (int64_t)t * a.qkv_stride + (int64_t)h * D + i0;
    lo = *reinterpret_cast<const uint4*>(row);
    hi = *reinterpret_cast<const uint4*>(row + D / 2);
    pos = a.positions[t];
    if (pos < 0 || pos >= a.max_pos) {
      if (live) set_device_error(kDevBadIndex);
      live = false;
      pos = 0;
    }
  };
  load(threadIdx.x);
  for (int base = 0; base < total; base += kAppendThreads) {  // uniform: the norm shuffles
    float x[16];
    unpack16(lo, hi, x);
    const Rope8 rp = load_rope<D>(a, pos, i0);
    const bool store = live;
    __nv_bfloat16* out = a.q_out + (int64_t)t * a.q_out_stride + (int64_t)h * D + i0;
    if (base + kAppendThreads < total) load(base + kAppendThreads + threadIdx.x);
    if (a.q_norm_w != nullptr) head_norm<D>(x, a.q_norm_w, i0, a.qk_eps, true);
    rotate16(x, rp);
    if (store) {
      uint4 l, g;
      l.x = pack_bf16x2(x[0], x[1]);
      l.y = pack_bf16x2(x[2], x[3]);
      l.z = pack_bf16x2(x[4], x[5]);
      l.w = pack_bf16x2(x[6], x[7]);
      g.x = pack_bf16x2(x[8], x[9]);
      g.y = pack_bf16x2(x[10], x[11]);
      g.z = pack_bf16x2(x[12], x[13]);
      g.w = pack_bf16x2(x[14], x[15]);
      *reinterpret_cast<uint4*>(out) = l;
      *reinterpret_cast<uint4*>(out + D / 2) = g;
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
  const int heads = kAppendThreads * 16 / (kKvBlock * head_dim);
  // Small steps are spread: a window's groups over as many CTAs, a q row a CTA, and rows
  // that are alone in their block get lanes of their own (a window would do 16 of them
  // one after the other: 29 us for 256 decode rows, and 6.3 so).  In large steps a CTA
  // keeps a window or 8 q rows and loads ahead: with a CTA for each group and q row, 8k
  // prompt rows took 61 us for 52.  Prompts change over evenly (1,024 rows 12.3 us, 1,025
  // 10.3); decode rows pay for it in a large step, whose windows take their rows one after
  // the other: 1,024 of them 12.4 us, 1,025 94, and 256 before 800 prompt rows 94.
  const bool large = num_tokens > 1024;
  a.groups = (2 * num_kv_heads + heads - 1) / heads;
  a.groups_per_cta = large ? a.groups : 1;
  a.group_ctas = (a.groups + a.groups_per_cta - 1) / a.groups_per_cta;
  a.q_tokens = large ? 8 : 1;
  const int64_t kv = (int64_t)((num_tokens + kWindow - 1) / kWindow) * a.group_ctas;
  const int64_t single = large ? 0
                               : ((int64_t)num_tokens * 2 * num_kv_heads * (head_dim / 16) +
                                  kAppendThreads - 1) / kAppendThreads;
  const int64_t q_ctas = (num_tokens + a.q_tokens - 1) / a.q_tokens;
  MUK_REQUIRE(kv + single + q_ctas <= INT32_MAX && (int64_t)num_q_heads * head_dim <= (1 << 24),
              "muk_rope_kv_append_fp8: %d tokens of %d heads", num_tokens, num_q_heads);
  a.kv_ctas = (int)kv;
  a.single_ctas = (int)single;
  const dim3 grid((unsigned)(kv + single + q_ctas));
  launch_pdl(head_dim == 128 ? rope_kv_append_fp8_kernel<128> : rope_kv_append_fp8_kernel<64>, grid,
             dim3(kAppendThreads), 0, as_stream(stream), a);
  return check_launch("muk_rope_kv_append_fp8");
}
