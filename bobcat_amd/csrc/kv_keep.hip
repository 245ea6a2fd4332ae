// The rows of the drafts that a step keeps, moved together behind the past.
//
// Position past + j gets the row of position past + path[j], j going up, in
// every layer's cache and KV head.  A path goes up, so path[j] >= j, and a place that
// was written is never read later; each thread owns one piece of all rows (16 bytes
// of the keys, an element of the values, a scale), so no thread reads what
// another writes.
#include "device.h"
#include "kernels.h"
#include "kv_cache.h"
#include "runtime.h"

namespace bch {

constexpr uint32_t kKeepBatch = 8;  // rows in flight

template <uint32_t FORMAT, uint32_t HD>
constexpr uint32_t keep_threads() {
  return (HD / (16 / kv_elem_bytes(FORMAT)) + HD + 2 + 63) / 64 * 64;
}

template <uint32_t FORMAT, uint32_t HD>
__global__ __launch_bounds__((keep_threads<FORMAT, HD>())) void k_kv_keep(KvGeometry g, uint64_t layer_bytes,
                                                                        const KvSeq *__restrict__ seqs,
                                                                        const uint32_t *__restrict__ kept,
                                                                        const uint32_t *__restrict__ path, uint32_t row0) {
  using Elem = std::conditional_t<FORMAT == BCH_KV_F16, uint16_t, uint8_t>;
  constexpr uint32_t E = 16 / sizeof(Elem), BYTES = kv_block_bytes(FORMAT, HD), PART = kKvBlock * HD * sizeof(Elem);
  constexpr uint32_t KEYS = HD / E, ALL = KEYS + HD + (FORMAT == BCH_KV_F16 ? 0 : 2);
  const KvSeq q = seqs[blockIdx.x];
  const uint32_t n = min(kept[blockIdx.x], q.n_new), head = blockIdx.y, t = threadIdx.x;
  path += q.row - row0;
  g.cache += blockIdx.z * layer_bytes;
  if (t >= ALL) return;
  auto block = [&](uint32_t at) {
    const uint32_t b = (q.past + at) / kKvBlock;
    return g.block<BYTES>(g.page(q.table, b), b, head);
  };
  // f(kind's type, offset in the block of position i)
  auto move = [&](auto type, auto offset) {
    using T = decltype(type);
    for (uint32_t j0 = 0; j0 < n; j0 += kKeepBatch) {
      T x[kKeepBatch];
      uint32_t from[kKeepBatch];
#pragma unroll
      for (uint32_t j = 0; j < kKeepBatch; j++) {
        const uint32_t p = j0 + j < n ? path[j0 + j] : 0;
        from[j] = p > j0 + j && p < q.n_new ? p : kKvNone;  // (the others are in place, or no path)
        if (from[j] != kKvNone) x[j] = *reinterpret_cast<const T *>(block(p) + offset((q.past + p) % kKvBlock));
      }
#pragma unroll
      for (uint32_t j = 0; j < kKeepBatch; j++)
        if (from[j] != kKvNone) *reinterpret_cast<T *>(block(j0 + j) + offset((q.past + j0 + j) % kKvBlock)) = x[j];
    }
  };
  if (t < KEYS)
    move(uint4{}, [&](uint32_t i) { return (t * kKvBlock + i) * 16; });
  else if (t < KEYS + HD)
    move(Elem{}, [&](uint32_t i) { return PART + kv_value_at<FORMAT>(i, t - KEYS) * (uint32_t)sizeof(Elem); });
  else
    move(float{}, [&](uint32_t i) { return 2 * PART + ((t - KEYS - HD) * kKvBlock + i) * 4; });
}

}  // namespace bch

using namespace bch;

extern "C" int bch_kv_keep(bch_ctx *ctx, const bch_kv_plan *plan, uint32_t first, uint32_t n_seqs, bch_view cache,
                           uint32_t n_layers, uint64_t layer_bytes, bch_view kept, bch_view path) {
  void *cp;
  uint32_t *np, *pp, row, tokens;
  BCH_TRY(kv_plan_cache(ctx, "kv_keep", plan, cache, &cp));
  BCH_TRY(kv_plan_range("kv_keep", plan, first, n_seqs, &row, &tokens));
  const bch_kv_shape &s = plan->shape;
  const uint64_t cache_bytes = bch_kv_page_bytes(&s) * s.n_pages;
  if (n_layers > 1) {
    if (layer_bytes < cache_bytes || layer_bytes % 16 || n_layers > 65535 || layer_bytes > (1ull << 48))
      return fail(BCH_ERR_ARGUMENT, "kv_keep: %u caches of %llu bytes %llu apart", n_layers, (unsigned long long)cache_bytes,
                  (unsigned long long)layer_bytes);
    BCH_TRY(check_view(ctx, "kv_keep", cache, layer_bytes * (n_layers - 1) + cache_bytes, &cp));
  }
  const uint64_t bytes = n_layers > 1 ? layer_bytes * (n_layers - 1) + cache_bytes : cache_bytes;
  BCH_TRY(view_ptr(ctx, "kv_keep", kept, (uint64_t)n_seqs * 4, &np));
  BCH_TRY(view_ptr(ctx, "kv_keep", path, (uint64_t)tokens * 4, &pp));
  if (reinterpret_cast<uintptr_t>(np) % 4 || reinterpret_cast<uintptr_t>(pp) % 4)
    return fail(BCH_ERR_ARGUMENT, "kv_keep: operands must be 4-byte aligned");
  if (kv_overlap(cp, bytes, np, (uint64_t)n_seqs * 4) || kv_overlap(cp, bytes, pp, (uint64_t)tokens * 4))
    return fail(BCH_ERR_ARGUMENT, "kv_keep: the path lies over the cache");
  return launch(ctx, {"kv_keep", n_seqs, s.n_kv_heads * s.head_dim, 0}, [&](hipStream_t st) {
    if (!tokens || !n_layers) return;
    kv_plan_use(ctx, plan);
    kv_dispatch(s.format, s.head_dim, [&](auto format, auto hd) {
      constexpr uint32_t F = decltype(format)::value, HD = decltype(hd)::value;
      k_kv_keep<F, HD><<<dim3(n_seqs, s.n_kv_heads, n_layers), keep_threads<F, HD>(), 0, st>>>(
          plan->geometry(cp), layer_bytes, plan->d_seqs + first, np, pp, row);
    });
  });
}
