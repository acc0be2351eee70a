// The KV-cache part of a decoder layer's step, shared by the native executors:
// where a layer's cache lies in the pool, and the append and attention entry
// points of its kind (bf16, or 8-bit codes with block scales).
#pragma once

#include <math.h>
#include <stdint.h>

#include "abi_util.h"

namespace muk {

// A layer's K and V caches; ks / vs are NULL for a bf16 pool.
struct KvLayer {
  void* k;
  void* v;
  float* ks;
  float* vs;
};

template <typename Model>
KvLayer kv_layer(const Model* m, int l) {
  const int64_t blocks = (int64_t)m->num_blocks * m->num_kv_heads;
  const int64_t bytes = blocks * m->block_size * m->head_dim * (m->kv_scales ? 1 : 2);
  auto* pool = static_cast<uint8_t*>(m->kv_pool);
  float* s = m->kv_scales;
  return {pool + 2 * l * bytes, pool + (2 * l + 1) * bytes, s ? s + 2 * l * blocks : nullptr,
          s ? s + (2 * l + 1) * blocks : nullptr};
}

// QK-norm (optional), RoPE and the KV append over a step's q|k|v rows, in place.
template <typename Model>
int kv_append(const Model* m, const MukStepBatch* b, const KvLayer& kv, const float* q_norm,
              const float* k_norm, void* stream) {
  const int Hq = m->num_q_heads, Hkv = m->num_kv_heads, D = m->head_dim;
  const int n = (Hq + 2 * Hkv) * D;
  if (kv.ks)
    return muk_rope_kv_append_fp8(m->qkv, n, m->qkv, n, b->positions, b->slot_mapping, m->rope_cos,
                                  m->rope_sin, m->rope_len, b->num_tokens, Hq, Hkv, D, q_norm,
                                  k_norm, 1e-6f, kv.k, kv.v, kv.ks, kv.vs, m->num_blocks,
                                  m->block_size, stream);
  return muk_rope_kv_append(m->qkv, n, b->positions, b->slot_mapping, m->rope_cos, m->rope_sin,
                            m->rope_len, b->num_tokens, Hq, Hkv, D, q_norm, k_norm, 1e-6f, kv.k,
                            kv.v, m->num_blocks, m->block_size, stream);
}

// Paged decode attention over the decode rows, varlen prefill attention over
// the rest (decode sequences own one row each, so prefill starts at num_decode).
// *launches (may be NULL) grows by the kernels launched.
template <typename Model>
int kv_attention(const Model* m, const MukStepBatch* b, const KvLayer& kv, int* launches,
                 void* stream) {
  const int B = b->num_seqs, nd = b->num_decode;
  const int Hq = m->num_q_heads, Hkv = m->num_kv_heads, D = m->head_dim;
  const int qkv_n = (Hq + 2 * Hkv) * D, attn_n = Hq * D;
  const float scale = 1.0f / sqrtf((float)D);
  const int bts = b->block_table_stride, bt_cap = bts * m->block_size;
  auto* qkv = static_cast<uint16_t*>(m->qkv);  // bf16, addressed in 2-byte elements
  auto* attn = static_cast<uint16_t*>(m->attn);
  if (nd > 0) {
    const int bound = b->decode_len_bound < bt_cap ? b->decode_len_bound : bt_cap;
    int rc;
    if (kv.ks)
      rc = muk_paged_decode_attn_fp8(qkv, qkv_n, attn, attn_n, kv.k, kv.v, kv.ks, kv.vs,
                                     b->block_tables, bts, b->seq_lens, nd, Hq, Hkv, D,
                                     m->block_size, m->num_blocks, scale, bound, m->attn_ws,
                                     m->attn_ws_bytes, stream);
    else
      rc = muk_paged_decode_attn(qkv, qkv_n, attn, attn_n, kv.k, kv.v, b->block_tables, bts,
                                 b->seq_lens, nd, Hq, Hkv, D, m->block_size, m->num_blocks, scale,
                                 bound, m->attn_ws, m->attn_ws_bytes, stream);
    if (rc != MUK_OK) return rc;
    if (launches) *launches += 2;
  }
  if (B > nd) {
    auto* q = qkv + (int64_t)nd * qkv_n;
    auto* out = attn + (int64_t)nd * attn_n;
    const int32_t* bt = b->block_tables + (int64_t)nd * bts;
    int rc;
    if (kv.ks)
      rc = muk_paged_prefill_attn_fp8(q, qkv_n, out, attn_n, kv.k, kv.v, kv.ks, kv.vs, bt, bts,
                                      b->seq_lens + nd, b->prefill_cu, B - nd, b->num_tokens - nd,
                                      b->max_q_len, bt_cap, Hq, Hkv, D, m->block_size,
                                      m->num_blocks, scale, stream);
    else
      rc = muk_paged_prefill_attn(q, qkv_n, out, attn_n, kv.k, kv.v, bt, bts, b->seq_lens + nd,
                                  b->prefill_cu, B - nd, b->max_q_len, Hq, Hkv, D, m->block_size,
                                  m->num_blocks, scale, stream);
    if (rc != MUK_OK) return rc;
    if (launches) *launches += 1;
  }
  return MUK_OK;
}

}  // namespace muk
