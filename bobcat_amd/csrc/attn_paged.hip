// Attention of a batch's new tokens over the paged cache: row i of a sequence
// with `past` positions attends to positions 0 .. past + i of its pages,
// softmax(q·k/√hd)·v with the keys and values that the cache holds (in the
// 8-bit formats scale·integer).
//
// One wave per token and query head: a lane scores one key of 64 at a time
// (the running maximum and sum of an online softmax), then owns every 64th
// element of the output.
#include <cmath>

#include "device.h"
#include "kernels.h"
#include "kv_cache.h"
#include "runtime.h"

namespace bch {

template <uint32_t FORMAT>
__device__ __forceinline__ float paged_float(const uint8_t *p) {
  if constexpr (FORMAT == BCH_KV_F16) return half_bits_to_float(*reinterpret_cast<const uint16_t *>(p));
  if constexpr (FORMAT == BCH_KV_I8) return (float)*reinterpret_cast<const int8_t *>(p);
  return __builtin_amdgcn_cvt_f32_fp8((int)*p, 0);
}

template <uint32_t FORMAT, uint32_t HD>
__global__ __launch_bounds__(64) void k_attn_paged(KvGeometry g, const KvSeq *__restrict__ seqs, uint32_t n_seqs,
                                                   const float *__restrict__ q, uint32_t q_stride, float *__restrict__ out,
                                                   uint32_t out_stride, uint32_t n_heads, float scale) {
  constexpr uint32_t BYTES = kv_block_bytes(FORMAT, HD), SIZE = kv_elem_bytes(FORMAT), PART = kKvBlock * HD * SIZE;
  __shared__ float q_s[HD], p_s[64];
  const uint32_t row = blockIdx.x, head = blockIdx.y, kv = head / (n_heads / g.n_kv), lane = threadIdx.x;
  uint32_t lo = 0, hi = n_seqs;  // the last sequence whose rows begin at or before this one (and that has rows)
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) / 2;
    if (seqs[mid].row <= row) lo = mid; else hi = mid;
  }
  const KvSeq seq = seqs[lo];
  const uint32_t n_keys = seq.past + (row - seq.row) + 1;
  for (uint32_t d = lane; d < HD; d += 64) q_s[d] = q[(uint64_t)row * q_stride + head * HD + d] * scale;
  float m = -INFINITY, l = 0.f, o[HD / 64];
  for (uint32_t j = 0; j < HD / 64; j++) o[j] = 0.f;
  __syncthreads();
  for (uint32_t t0 = 0; t0 < n_keys; t0 += 64) {
    const uint32_t key = t0 + lane, len = min(64u, n_keys - t0);
    float s = -INFINITY;
    if (lane < len) {
      const uint8_t *block = g.block<BYTES>(seq.table, key / kKvBlock, kv);
      s = 0.f;
      for (uint32_t d = 0; d < HD; d++) s = fmaf(q_s[d], paged_float<FORMAT>(block + kv_key_at<FORMAT>(key % kKvBlock, d) * SIZE), s);
      if constexpr (FORMAT != BCH_KV_F16) s *= reinterpret_cast<const float *>(block + 2 * PART)[key % kKvBlock];
    }
    // (A NaN score passes the maximum by and makes the sum NaN.)
    const float m_new = fmaxf(m, wave_max(s)), m_use = m_new == -INFINITY ? 0.f : m_new;
    const float p = lane < len ? expf(s - m_use) : 0.f;
    const float corr = expf(m - m_use);
    l = l * corr + wave_sum(p);
    m = m_new;
    __syncthreads();
    p_s[lane] = p;
    __syncthreads();
    for (uint32_t j = 0; j < HD / 64; j++) {
      const uint32_t d = lane + 64 * j;
      float a = o[j] * corr;
      for (uint32_t i = 0; i < len; i++) {
        const uint8_t *block = g.block<BYTES>(seq.table, (t0 + i) / kKvBlock, kv);
        float x = paged_float<FORMAT>(block + PART + kv_value_at<FORMAT>((t0 + i) % kKvBlock, d) * SIZE);
        if constexpr (FORMAT != BCH_KV_F16) x *= reinterpret_cast<const float *>(block + 2 * PART)[kKvBlock + (t0 + i) % kKvBlock];
        a = fmaf(p_s[i], x, a);
      }
      o[j] = a;
    }
  }
  for (uint32_t j = 0; j < HD / 64; j++) out[(uint64_t)row * out_stride + head * HD + lane + 64 * j] = o[j] / l;
}

}  // namespace bch

using namespace bch;

extern "C" int bch_attention_paged(bch_ctx *ctx, const bch_kv_plan *plan, bch_view cache, bch_view q, uint32_t q_stride,
                                   bch_view out, uint32_t out_stride) {
  void *cp;
  float *qp, *op;
  BCH_TRY(kv_plan_cache(ctx, "attention_paged", plan, cache, &cp));
  const bch_kv_shape &s = plan->shape;
  const uint32_t width = plan->n_heads * s.head_dim;
  BCH_TRY(kv_plan_rows(ctx, "attention_paged", plan, q, width, q_stride, &qp));
  BCH_TRY(kv_plan_rows(ctx, "attention_paged", plan, out, width, out_stride, &op));
  const uint64_t out_bytes = kv_rows_bytes(plan, width, out_stride);
  if (kv_overlap(cp, bch_kv_page_bytes(&s) * s.n_pages, op, out_bytes))
    return fail(BCH_ERR_ARGUMENT, "attention_paged: the outputs lie over the cache");
  if (kv_overlap(qp, kv_rows_bytes(plan, width, q_stride), op, out_bytes)) {
    // Side by side in rows of one stride they may lie.
    const uint64_t apart = qp < op ? (uint64_t)(op - qp) % q_stride : q_stride - (uint64_t)(qp - op) % q_stride;
    if (q_stride != out_stride || apart < width || apart > q_stride - width)
      return fail(BCH_ERR_ARGUMENT, "attention_paged: the outputs lie over the queries");
  }
  return launch(ctx, {"attention_paged", plan->n_tokens, width, 0}, [&](hipStream_t st) {
    if (!plan->n_tokens) return;
    kv_dispatch(s.format, s.head_dim, [&](auto format, auto hd) {
      k_attn_paged<decltype(format)::value, decltype(hd)::value><<<dim3(plan->n_tokens, plan->n_heads), 64, 0, st>>>(
          plan->geometry(cp), plan->d_seqs, plan->n_seqs, qp, q_stride, op, out_stride, plan->n_heads,
          1.0f / sqrtf((float)s.head_dim));
    });
  });
}
