// The rows of the drafts that a step keeps, moved together behind the past.
//
// Position past + j gets the row of position past + path[j], j going up, in
// every layer's cache and KV head.  A path goes up, so path[j] >= j: of the rows in one
// batch all are read before one is written, and a place that was written is never
// read by a later batch.
//
// Bound by latency: the path, the pages, the rows.  So a workgroup looks its
// sequence's pages up once, a lane a row, for a few heads and layers, and brings
// all their pieces at once (64 sequences, 2 or 3 rows each, eight heads of 64 and eight layers of
// int8: 5.6 us; a thread for each piece of one head and layer, the rows in turn, 13.2).
#include "device.h"
#include "kernels.h"
#include "kv_cache.h"
#include "runtime.h"

namespace bch {

constexpr uint32_t kKeepThreads = 256, kKeepRows = 8;  // rows of a batch
// Heads of layers that a workgroup does: as many as give each thread eight elements of values.
constexpr uint32_t keep_pairs(uint32_t hd) { return 256 / hd; }

template <uint32_t FORMAT, uint32_t HD>
__global__ __launch_bounds__(kKeepThreads) void k_kv_keep(KvGeometry g, uint64_t layer_bytes, uint32_t n_pairs,
                                                          const KvSeq *__restrict__ seqs,
                                                          const uint32_t *__restrict__ kept,
                                                          const uint32_t *__restrict__ path, uint32_t row0) {
  using Elem = std::conditional_t<FORMAT == BCH_KV_F16, uint16_t, uint8_t>;
  constexpr uint32_t E = 16 / sizeof(Elem), BYTES = kv_block_bytes(FORMAT, HD), PART = kKvBlock * HD * sizeof(Elem);
  constexpr uint32_t PAIRS = keep_pairs(HD), KEYS = HD / E, PER = PAIRS * kKeepRows * HD / kKeepThreads;
  static_assert(PAIRS * kKeepRows * KEYS <= kKeepThreads);
  struct Move {
    uint64_t from, to;  // blocks of head 0
    uint32_t i, j;      // positions in them
  };
  __shared__ Move moves_s[kKeepRows];
  const KvSeq q = seqs[blockIdx.x];
  const uint32_t n = min(kept[blockIdx.x], q.n_new), tid = threadIdx.x;
  path += q.row - row0;
  const uint32_t pair0 = blockIdx.y * PAIRS, pairs = min(PAIRS, n_pairs - pair0);
  // Head pair % n_kv of layer pair / n_kv.
  auto base = [&](uint32_t pair) {
    const uint32_t layer = (pair0 + pair) / g.n_kv, head = (pair0 + pair) % g.n_kv;
    return g.cache + layer * layer_bytes + (uint64_t)head * g.page_blocks * BYTES;
  };
  for (uint32_t j0 = 0; j0 < n; j0 += kKeepRows) {
    // The batch's rows that move, one behind the other.
    uint32_t count = 0;
    {
      const uint32_t lane = tid % 64, to = j0 + lane, from = lane < kKeepRows && to < n ? path[to] : 0;
      const bool moves = from > to && from < q.n_new;  // (the others are in place, or no path)
      const uint64_t all = __builtin_amdgcn_ballot_w64(moves);
      count = __popcll(all);
      if (tid < 64 && moves) {
        auto place = [&](uint32_t at, uint32_t *i) {
          const uint32_t p = q.past + at, b = p / kKvBlock;
          *i = p % kKvBlock;
          return ((uint64_t)g.page(q.table, b) * g.n_kv * g.page_blocks + g.in_page(b)) * BYTES;
        };
        Move m;
        m.from = place(from, &m.i);
        m.to = place(to, &m.j);
        moves_s[__popcll(all & ((1ull << lane) - 1))] = m;
      }
    }
    __syncthreads();
    // Piece `piece` of row r of head and layer `pair`: items in this order, the rows slowest.
    uint4 key;
    Elem value[PER];
    float scale;
    const uint32_t key_rp = tid / KEYS, scale_rp = tid / 2;
    const bool has_key = key_rp < count * PAIRS && key_rp % PAIRS < pairs;
    const bool has_scale = FORMAT != BCH_KV_F16 && scale_rp < count * PAIRS && scale_rp % PAIRS < pairs;
    auto key_at = [&](uint64_t block, uint32_t i) {
      return reinterpret_cast<uint4 *>(base(key_rp % PAIRS) + block + (tid % KEYS * kKvBlock + i) * 16);
    };
    auto scale_at = [&](uint64_t block, uint32_t i) {
      return reinterpret_cast<float *>(base(scale_rp % PAIRS) + block + 2 * PART + (tid % 2 * kKvBlock + i) * 4);
    };
    auto value_at = [&](uint32_t k, uint64_t block, uint32_t i) {
      const uint32_t item = k * kKeepThreads + tid, pair = item / HD % PAIRS, d = item % HD;
      return reinterpret_cast<Elem *>(base(pair) + block + PART) + kv_value_at<FORMAT>(i, d);
    };
    auto has_value = [&](uint32_t k) {
      const uint32_t rp = (k * kKeepThreads + tid) / HD;
      return rp < count * PAIRS && rp % PAIRS < pairs;
    };
    if (has_key) key = *key_at(moves_s[key_rp / PAIRS].from, moves_s[key_rp / PAIRS].i);
#pragma unroll
    for (uint32_t k = 0; k < PER; k++) {
      const Move &m = moves_s[(k * kKeepThreads + tid) / (HD * PAIRS)];
      if (has_value(k)) value[k] = *value_at(k, m.from, m.i);
    }
    if (has_scale) scale = *scale_at(moves_s[scale_rp / PAIRS].from, moves_s[scale_rp / PAIRS].i);
    __builtin_amdgcn_s_waitcnt(0);  // all rows of the batch are read before one is written
    __syncthreads();
    if (has_key) *key_at(moves_s[key_rp / PAIRS].to, moves_s[key_rp / PAIRS].j) = key;
#pragma unroll
    for (uint32_t k = 0; k < PER; k++) {
      const Move &m = moves_s[(k * kKeepThreads + tid) / (HD * PAIRS)];
      if (has_value(k)) *value_at(k, m.to, m.j) = value[k];
    }
    if (has_scale) *scale_at(moves_s[scale_rp / PAIRS].to, moves_s[scale_rp / PAIRS].j) = scale;
    __syncthreads();  // the next batch's rows come to the same place, and read behind these
  }
}

}  // namespace bch

using namespace bch;

extern "C" int bch_kv_keep(bch_ctx *ctx, const bch_kv_plan *plan, uint32_t first, uint32_t n_seqs, bch_view cache,
                           uint32_t n_layers, uint64_t layer_bytes, bch_view kept, bch_view path) {
  void *cp;
  uint32_t *np, *pp, row, tokens;
  BCH_TRY(kv_plan_cache(ctx, "kv_keep", plan, cache, &cp));
  BCH_TRY(kv_plan_range("kv_keep", plan, first, n_seqs, &row, &tokens));
  // (A workgroup of 256 threads for each: a launch has fewer than 2^32.)
  if (n_seqs >= 1u << 24) return fail(BCH_ERR_ARGUMENT, "kv_keep: %u sequences", n_seqs);
  const bch_kv_shape &s = plan->shape;
  const uint64_t cache_bytes = bch_kv_page_bytes(&s) * s.n_pages;
  if (n_layers > 1) {
    if (layer_bytes < cache_bytes || layer_bytes % 16 || n_layers > 128 || layer_bytes > (1ull << 48))
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
      const uint32_t pairs = s.n_kv_heads * n_layers;
      k_kv_keep<F, HD><<<dim3(n_seqs, div_ceil(pairs, keep_pairs(HD))), kKeepThreads, 0, st>>>(
          plan->geometry(cp), layer_bytes, pairs, plan->d_seqs + first, np, pp, row);
    });
  });
}
