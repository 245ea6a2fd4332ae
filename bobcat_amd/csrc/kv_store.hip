// Keys and values quantised into the pages of a cache as a batch brings them,
// and read back as floats.
//
// A row x of hd floats (one position and KV head) is kept as f16, or as
// y = clamp(x / s, -top, top) rounded to int8 (top 127) or e4m3 (top 448) with
// the row's own scale s = clamp(max|x|·(1/top), 2^-40, 2^60), 1/top rounded to
// f32; it reads back as s·y.  A row that holds a NaN or an infinity gets the
// scale NaN, so all of it reads back as NaN.
//
// Both are one pass over the floats, a workgroup for every block of 16 positions
// and KV head, and bound by their bytes where there are many (6,400 new
// tokens, 8 heads of 128 into e4m3: 14.8 us, 4.4 TB/s; 30,000 positions of 8
// heads of 64 out of int8: 33.9 us, 4.6 TB/s), else by a launch's latency (eight
// tokens 2.9 us).
#include <cmath>

#include "device.h"
#include "kernels.h"
#include "kv_cache.h"
#include "runtime.h"

namespace bch {

constexpr uint32_t kStoreThreads = 256;  // 16 lanes for each of a block's 16 rows

// The scale of a row from the largest magnitude of its elements, of which one
// that is not finite counts as infinite.
__device__ __forceinline__ float kv_scale(float largest, float top) {
  const float s = fminf(fmaxf(largest * (1.f / top), kKvScaleMin), kKvScaleMax);
  return largest <= 3.402823466e38f ? s : __int_as_float(0x7fc00000);
}

// Four elements of a row as the cache's bytes (f16: two dwords).  The quotients
// are IEEE divisions: the stored values are those of the definition, bit for
// bit.  A row of scale NaN is kept as zeros.
template <uint32_t FORMAT>
__device__ __forceinline__ uint2 kv_quantise(float4 x, float s) {
  if constexpr (FORMAT == BCH_KV_F16) {
    const __half2 a = __floats2half2_rn(x.x, x.y), b = __floats2half2_rn(x.z, x.w);
    return {*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b)};
  } else {
    constexpr float top = FORMAT == BCH_KV_I8 ? 127.f : 448.f;
    const bool fine = s == s;
    const float v[4] = {x.x, x.y, x.z, x.w};
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; i++) y[i] = fine ? fminf(fmaxf(v[i] / s, -top), top) : 0.f;
    if constexpr (FORMAT == BCH_KV_I8) {
      uint32_t w = 0;
#pragma unroll
      for (int i = 0; i < 4; i++) w |= ((uint32_t)(int)rintf(y[i]) & 0xffu) << (8 * i);
      return {w, 0};
    } else {
      int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
      w = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
      return {(uint32_t)w, 0};
    }
  }
}

// Element `i` (0..3) of four from kv_quantise.
template <uint32_t FORMAT>
__device__ __forceinline__ uint32_t kv_element(uint2 w, int i) {
  if constexpr (FORMAT == BCH_KV_F16) return ((i < 2 ? w.x : w.y) >> (16 * (i & 1))) & 0xffffu;
  return (w.x >> (8 * i)) & 0xffu;
}

template <uint32_t FORMAT, uint32_t HD>
__global__ __launch_bounds__(kStoreThreads) void k_kv_store(const KvStoreItem *__restrict__ items, KvGeometry g,
                                                            const float *__restrict__ k, uint32_t k_stride,
                                                            const float *__restrict__ v, uint32_t v_stride) {
  using Elem = std::conditional_t<FORMAT == BCH_KV_F16, uint16_t, uint8_t>;
  constexpr uint32_t J = HD / 64, BYTES = kv_block_bytes(FORMAT, HD), PART = kKvBlock * HD * sizeof(Elem);
  __shared__ __align__(16) Elem v_s[kKvBlock * HD];
  const KvStoreItem it = items[blockIdx.x];
  const uint32_t head = blockIdx.y, r = threadIdx.x / 16, c = threadIdx.x % 16, pos = it.pos % kKvBlock + r;
  uint8_t *const block = g.block<BYTES>(it.page, it.pos / kKvBlock, head);
  const bool mine = r < it.n;
  const uint64_t row = it.row + (mine ? r : 0);
  float4 x[2][J];
  float largest[2] = {0.f, 0.f};
#pragma unroll
  for (int t = 0; t < 2; t++) {
    const float *src = (t ? v + row * v_stride : k + row * k_stride) + (uint64_t)head * HD + 4 * c;
#pragma unroll
    for (uint32_t j = 0; j < J; j++) x[t][j] = *reinterpret_cast<const float4 *>(src + 64 * j);
  }
  float scale[2] = {1.f, 1.f};
  if constexpr (FORMAT != BCH_KV_F16) {
#pragma unroll
    for (int t = 0; t < 2; t++) {
#pragma unroll
      for (uint32_t j = 0; j < J; j++) {
        const float e[4] = {x[t][j].x, x[t][j].y, x[t][j].z, x[t][j].w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float a = fabsf(e[i]);
          largest[t] = fmaxf(largest[t], a <= 3.402823466e38f ? a : INFINITY);
        }
      }
      // Over the row's 16 lanes.
      largest[t] = fmaxf(largest[t], dpp<kDppXor1>(largest[t]));
      largest[t] = fmaxf(largest[t], dpp<kDppXor2>(largest[t]));
      largest[t] = fmaxf(largest[t], dpp<kDppHalfMirror>(largest[t]));
      largest[t] = fmaxf(largest[t], dpp<kDppMirror>(largest[t]));
      scale[t] = kv_scale(largest[t], FORMAT == BCH_KV_I8 ? 127.f : 448.f);
    }
    if (mine && c < 2) reinterpret_cast<float *>(block + 2 * PART)[c * kKvBlock + pos] = scale[c];
  }
  // A whole block's values cross in LDS and leave in pieces of 16 bytes; the
  // rows of a part are stored element by element, so that the block's other
  // positions keep their bytes.
  const bool whole = it.n == kKvBlock;
  Elem *const keys = reinterpret_cast<Elem *>(block), *const values = reinterpret_cast<Elem *>(block + PART);
#pragma unroll
  for (uint32_t j = 0; j < J; j++) {
    const uint32_t d = 64 * j + 4 * c;
    const uint2 kq = kv_quantise<FORMAT>(x[0][j], scale[0]), vq = kv_quantise<FORMAT>(x[1][j], scale[1]);
    if (mine) {
      if constexpr (FORMAT == BCH_KV_F16)
        *reinterpret_cast<uint2 *>(keys + kv_key_at<FORMAT>(pos, d)) = kq;
      else
        *reinterpret_cast<uint32_t *>(keys + kv_key_at<FORMAT>(pos, d)) = kq.x;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const Elem e = (Elem)kv_element<FORMAT>(vq, i);
      if (whole)
        v_s[kv_value_at<FORMAT>(r, d + i)] = e;
      else if (mine)
        values[kv_value_at<FORMAT>(pos, d + i)] = e;
    }
  }
  if (!whole) return;
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < PART / 16; i += kStoreThreads)
    reinterpret_cast<uint4 *>(values)[i] = reinterpret_cast<const uint4 *>(v_s)[i];
}

// One element as a float, without its scale.
template <uint32_t FORMAT>
__device__ __forceinline__ float kv_float(uint32_t bits) {
  if constexpr (FORMAT == BCH_KV_F16) return half_bits_to_float(bits);
  if constexpr (FORMAT == BCH_KV_I8) return (float)(int8_t)bits;
  return __builtin_amdgcn_cvt_f32_fp8((int)bits, 0);
}

// Positions first .. first + n of one sequence: a workgroup per block and head
// brings the block into LDS, and 16 lanes write each row.
template <uint32_t FORMAT, uint32_t HD>
__global__ __launch_bounds__(kStoreThreads) void k_kv_load(KvGeometry g, uint32_t table, uint32_t first, uint32_t n,
                                                           float *__restrict__ k, float *__restrict__ v) {
  using Elem = std::conditional_t<FORMAT == BCH_KV_F16, uint16_t, uint8_t>;
  constexpr uint32_t J = HD / 64, BYTES = kv_block_bytes(FORMAT, HD), PART = kKvBlock * HD * sizeof(Elem);
  __shared__ __align__(16) uint8_t s[BYTES];
  const uint32_t b = first / kKvBlock + blockIdx.x, head = blockIdx.y;
  const uint8_t *block = g.block<BYTES>(g.page(table, b), b, head);
  for (uint32_t i = threadIdx.x; i < BYTES / 16; i += kStoreThreads)
    reinterpret_cast<uint4 *>(s)[i] = reinterpret_cast<const uint4 *>(block)[i];
  __syncthreads();
  const uint32_t r = threadIdx.x / 16, c = threadIdx.x % 16, pos = b * kKvBlock + r;
  if (pos < first || pos - first >= n) return;
  const Elem *keys = reinterpret_cast<const Elem *>(s), *values = reinterpret_cast<const Elem *>(s + PART);
  float scale[2] = {1.f, 1.f};
  if constexpr (FORMAT != BCH_KV_F16) {
    scale[0] = reinterpret_cast<const float *>(s + 2 * PART)[r];
    scale[1] = reinterpret_cast<const float *>(s + 2 * PART)[kKvBlock + r];
  }
  const uint64_t out = ((uint64_t)(pos - first) * g.n_kv + head) * HD;
#pragma unroll
  for (uint32_t j = 0; j < J; j++) {
    const uint32_t d = 64 * j + 4 * c;
    float a[4], b4[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      a[i] = kv_float<FORMAT>(keys[kv_key_at<FORMAT>(r, d + i)]) * scale[0];
      b4[i] = kv_float<FORMAT>(values[kv_value_at<FORMAT>(r, d + i)]) * scale[1];
    }
    *reinterpret_cast<float4 *>(k + out + d) = float4{a[0], a[1], a[2], a[3]};
    *reinterpret_cast<float4 *>(v + out + d) = float4{b4[0], b4[1], b4[2], b4[3]};
  }
}

}  // namespace bch

using namespace bch;

extern "C" int bch_kv_store(bch_ctx *ctx, const bch_kv_plan *plan, bch_view cache, bch_view k, uint32_t k_stride,
                            bch_view v, uint32_t v_stride) {
  void *cp;
  float *kp, *vp;
  BCH_TRY(kv_plan_cache(ctx, "kv_store", plan, cache, &cp));
  const bch_kv_shape &s = plan->shape;
  const uint32_t width = s.n_kv_heads * s.head_dim;
  BCH_TRY(kv_plan_rows(ctx, "kv_store", plan, k, width, k_stride, &kp));
  BCH_TRY(kv_plan_rows(ctx, "kv_store", plan, v, width, v_stride, &vp));
  const uint64_t cache_bytes = bch_kv_page_bytes(&s) * s.n_pages;
  if (kv_overlap(cp, cache_bytes, kp, kv_rows_bytes(plan, width, k_stride)) ||
      kv_overlap(cp, cache_bytes, vp, kv_rows_bytes(plan, width, v_stride)))
    return fail(BCH_ERR_ARGUMENT, "kv_store: the rows lie over the cache");
  return launch(ctx, {"kv_store", plan->n_tokens, width, 0}, [&](hipStream_t st) {
    if (!plan->n_store) return;
    kv_plan_use(ctx, plan);
    kv_dispatch(s.format, s.head_dim, [&](auto format, auto hd) {
      k_kv_store<decltype(format)::value, decltype(hd)::value><<<dim3(plan->n_store, s.n_kv_heads), kStoreThreads, 0, st>>>(
          plan->d_store, plan->geometry(cp), kp, k_stride, vp, v_stride);
    });
  });
}

extern "C" int bch_kv_load(bch_ctx *ctx, const bch_kv_plan *plan, bch_view cache, uint32_t seq, uint32_t first,
                           uint32_t n, bch_view k, bch_view v) {
  void *cp;
  float *kp, *vp;
  BCH_TRY(kv_plan_cache(ctx, "kv_load", plan, cache, &cp));
  const bch_kv_shape &s = plan->shape;
  if (seq >= plan->n_seqs) return fail(BCH_ERR_ARGUMENT, "kv_load: sequence %u of %u", seq, plan->n_seqs);
  const KvSeq &q = plan->seqs[seq];
  if ((uint64_t)first + n > (uint64_t)q.past + q.n_new)
    return fail(BCH_ERR_OUT_OF_BOUNDS, "kv_load: positions up to %llu of a sequence of %u",
                (unsigned long long)first + n, q.past + q.n_new);
  const uint64_t bytes = (uint64_t)n * s.n_kv_heads * s.head_dim * 4;
  BCH_TRY(view_ptr(ctx, "kv_load", k, bytes, &kp));
  BCH_TRY(view_ptr(ctx, "kv_load", v, bytes, &vp));
  if (reinterpret_cast<uintptr_t>(kp) % 16 || reinterpret_cast<uintptr_t>(vp) % 16)
    return fail(BCH_ERR_ARGUMENT, "kv_load: rows must be 16-byte aligned");
  const uint64_t cache_bytes = bch_kv_page_bytes(&s) * s.n_pages;
  if (kv_overlap(cp, cache_bytes, kp, bytes) || kv_overlap(cp, cache_bytes, vp, bytes) || kv_overlap(kp, bytes, vp, bytes))
    return fail(BCH_ERR_ARGUMENT, "kv_load: the keys, the values and the cache lie over each other");
  return launch(ctx, {"kv_load", n, s.n_kv_heads * s.head_dim, 0}, [&](hipStream_t st) {
    if (!n) return;
    kv_plan_use(ctx, plan);
    const uint32_t blocks = (first + n - 1) / kKvBlock - first / kKvBlock + 1;
    kv_dispatch(s.format, s.head_dim, [&](auto format, auto hd) {
      k_kv_load<decltype(format)::value, decltype(hd)::value><<<dim3(blocks, s.n_kv_heads), kStoreThreads, 0, st>>>(
          plan->geometry(cp), q.table, first, n, kp, vp);
    });
  });
}
