// The paged key/value cache: the blocks' layout and what a plan holds
// (kv_plan.hip), shared by the kernels that write, read back and attend to it.
//
// A page holds page_size positions of every KV head, head after head; a
// head's part is one block for every 16 positions: the 16 keys, the 16 values
// and, in the 8-bit formats, their 16 + 16 f32 scales.  Within a block both
// lie as the matrix instructions take them, so that every load of a wave is
// one contiguous KB and no kernel transposes what it reads:
//   keys:   pieces of 16 bytes (E elements of a key), [piece][key];
//   values: pieces of 16 bytes, [64 (f16: 32) elements][quad of keys]
//           [element % 16][element / 16][key of the quad].
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>
#include <vector>

#include "../../include/bobcat_hip.h"

namespace bch {

constexpr uint32_t kKvBlock = 16;         // positions of a block
constexpr uint32_t kKvMaxPage = 512;      // positions of a page, at most
constexpr uint32_t kKvMaxGroup = 32;      // query heads per KV head, at most

// Scales are kept inside these, so that products of scales, and their
// reciprocals, stay far from f32's ends.
constexpr float kKvScaleMin = 0x1p-40f, kKvScaleMax = 0x1p60f;

__host__ __device__ constexpr uint32_t kv_elem_bytes(uint32_t format) { return format == BCH_KV_F16 ? 2 : 1; }
__host__ __device__ constexpr uint32_t kv_block_bytes(uint32_t format, uint32_t hd) {
  return 2 * kKvBlock * hd * kv_elem_bytes(format) + (format == BCH_KV_F16 ? 0 : 2 * kKvBlock * 4);
}
// Offsets, in elements from the start of the block's keys and of its values,
// of element d of position i.
template <uint32_t FORMAT>
__device__ __forceinline__ uint32_t kv_key_at(uint32_t i, uint32_t d) {
  constexpr uint32_t E = 16 / kv_elem_bytes(FORMAT);
  return (d / E * kKvBlock + i) * E + d % E;
}
template <uint32_t FORMAT>
__device__ __forceinline__ uint32_t kv_value_at(uint32_t i, uint32_t d) {
  constexpr uint32_t M = 4 / kv_elem_bytes(FORMAT);
  return (((d / (16 * M) * 4 + i / 4) * 16 + d % 16) * M + d / 16 % M) * 4 + i % 4;
}

// f(format, hd) with both as integral constants; the shape has been checked.
template <class F>
void kv_dispatch(uint32_t format, uint32_t hd, F &&f) {
  auto with_hd = [&](auto fmt) {
    if (hd == 64)
      f(fmt, std::integral_constant<uint32_t, 64>{});
    else if (hd == 128)
      f(fmt, std::integral_constant<uint32_t, 128>{});
    else
      f(fmt, std::integral_constant<uint32_t, 256>{});
  };
  if (format == BCH_KV_F16)
    with_hd(std::integral_constant<uint32_t, BCH_KV_F16>{});
  else if (format == BCH_KV_I8)
    with_hd(std::integral_constant<uint32_t, BCH_KV_I8>{});
  else
    with_hd(std::integral_constant<uint32_t, BCH_KV_F8>{});
}

// What the kernels know of a plan.
struct KvSeq {
  uint32_t past, n_new;  // positions before this batch's tokens, and the tokens
  uint32_t row;          // of the first token among the batch's
  uint32_t table;        // of the first page among the batch's pages
};
// New tokens that go into one block: their rows in the batch, and the place of
// the first among its sequence's positions.
struct KvStoreItem {
  uint32_t page, pos, row, n;
};
constexpr uint32_t kKvNone = ~0u;
// A new token of a batch with trees: the places of its parent, its first child
// and its parent's next child among its sequence's new tokens (kKvNone: none), its
// position, and where its mask begins (kKvNone: its sequence is a chain).
struct KvNode {
  uint32_t parent, child, sibling, position, mask;
};
// The mask of a tree's token: a bit for each key that it sees from key
// past / 32·32 on, 32 keys a word, to the word with the sequence's last.
__host__ __device__ constexpr uint32_t kv_mask_words(uint32_t past, uint32_t n_new) {
  return (past + n_new - 1) / 32 - past / 32 + 1;
}
// A tile of packed rows (row = token·group + head of the group) of a sequence
// and a part of its keys.
struct KvAttnItem {
  uint32_t table, past, row;  // of the sequence (KvSeq)
  uint32_t first, rows;       // packed rows first .. first + rows
  uint32_t lo, hi;            // steps of 32 keys
  uint32_t part;              // the first of its n_kv·rows records, ~0: writes the outputs itself
};
// The tiles whose keys are split, with the first split's records.
struct KvJoinItem {
  uint32_t row, first, rows, splits, part;
};
// Items dealt to workgroups: workgroup w of a KV head takes items starts[w] ..
// starts[w + 1].  (Where each has one, the kernels get no starts and save a
// load that the item's own load would wait for.)
struct KvWork {
  std::vector<KvAttnItem> items;
  std::vector<uint32_t> starts;
};
struct KvSchedule {
  KvWork tiles8, tiles16, chunks;  // tiles of at most 8, at most 16, and up to 128 rows
  std::vector<KvJoinItem> join;
  uint64_t records = 0;
  uint32_t tree_blocks = 0;  // of 16 rows, of tiles16 at most where there are trees
};
// attn_paged.hip: the attention's work of a batch, with no more partial
// results than partial_floats hold; with `trees` for the kernels of attn_tree.hip.
KvSchedule kv_schedule(const std::vector<KvSeq> &seqs, uint32_t group, uint32_t n_kv, uint32_t format, uint32_t head_dim,
                       uint32_t n_cus, uint64_t partial_floats, bool trees);

struct KvGeometry {
  uint8_t *cache;
  const uint32_t *pages;
  uint32_t n_kv, page_blocks;  // blocks of a page and head
  uint32_t page_magic;         // ceil(2^31 / page_blocks)
  // Block b of a sequence whose pages start at `table`: its page, by a scalar
  // load where both are uniform (the pages are constant while a kernel runs),
  // and its address for KV head `head`.  (The quotient is exact for b < 2^26 and
  // page_blocks <= 32.)
  __device__ __forceinline__ uint32_t page(uint32_t table, uint32_t b) const {
    using Constant = const __attribute__((address_space(4))) uint32_t;
    return ((Constant *)pages)[table + __umulhi(2 * b, page_magic)];
  }
  __device__ __forceinline__ uint32_t in_page(uint32_t b) const { return b - __umulhi(2 * b, page_magic) * page_blocks; }
  template <uint32_t BYTES>
  __device__ __forceinline__ uint8_t *block(uint32_t page, uint32_t b, uint32_t head) const {
    const uint32_t in_page = this->in_page(b);
    return cache + (((uint64_t)page * n_kv + head) * page_blocks + in_page) * BYTES;
  }
};

}  // namespace bch

// A batch's sequences and pages, checked and laid out for the kernels.
struct bch_kv_plan {
  bch_ctx *ctx;
  bch_kv_shape shape;
  uint32_t n_heads;
  bool ready = false;  // bch_kv_plan_set has succeeded
  // The last recording whose launches read the plan's memory (bch_ctx::begun).
  mutable uint64_t last_use = 0;
  uint32_t n_seqs = 0, n_tokens = 0;
  std::vector<bch::KvSeq> seqs;
  std::vector<uint8_t> rooted;  // sequences whose first new token is all others' ancestor; none: all of them
  const bch::KvSeq *d_seqs = nullptr;
  // One device allocation with all of the below, grown on demand.
  uint8_t *memory = nullptr;
  uint64_t memory_bytes = 0;
  const uint32_t *d_pages = nullptr;
  const bch::KvStoreItem *d_store = nullptr;
  uint32_t n_store = 0;
  // A batch with trees (else null): a node for each new token, and the masks.
  const bch::KvNode *d_nodes = nullptr;
  const uint32_t *d_masks = nullptr;
  uint32_t tree_blocks = 0;  // (KvSchedule)
  struct Work {
    const bch::KvAttnItem *items = nullptr;
    const uint32_t *starts = nullptr;
    uint32_t groups = 0;  // workgroups for each KV head
  } tiles8, tiles16, chunks;
  const bch::KvJoinItem *d_join = nullptr;
  uint32_t n_join = 0, join_rows = 0, join_splits = 0;  // the most rows and splits of a joined tile

  bch::KvGeometry geometry(void *cache) const {
    const uint32_t blocks = shape.page_size / bch::kKvBlock;
    return {static_cast<uint8_t *>(cache), d_pages, shape.n_kv_heads, blocks,
            ((1u << 31) + blocks - 1) / blocks};
  }
};

namespace bch {
// The plan of a recorded op: BCH_OK if it belongs to ctx and is ready.
int kv_plan_ready(bch_ctx *ctx, const char *kernel, const bch_kv_plan *plan);
// The same, and the view `cache` holds its pages, whose address goes to *ptr.
int kv_plan_cache(bch_ctx *ctx, const char *kernel, const bch_kv_plan *plan, bch_view cache, void **ptr);
// Notes that the open recording has launches that read the plan's memory.
void kv_plan_use(const bch_ctx *ctx, const bch_kv_plan *plan);
// Rows of `width` floats, `stride` apart, one for each of the plan's tokens.
int kv_plan_rows(bch_ctx *ctx, const char *kernel, const bch_kv_plan *plan, bch_view view, uint32_t width,
                 uint32_t stride, float **ptr);
// The bytes from a row's first float to the last row's end.
inline uint64_t kv_rows_bytes(const bch_kv_plan *plan, uint32_t width, uint32_t stride) {
  return plan->n_tokens ? ((uint64_t)(plan->n_tokens - 1) * stride + width) * 4 : 0;
}
// Sequences first .. first + n of a plan that has a batch, and their new tokens.
int kv_plan_range(const char *kernel, const bch_kv_plan *plan, uint32_t first, uint32_t n, uint32_t *row, uint32_t *tokens);
inline bool kv_overlap(const void *a, uint64_t a_bytes, const void *b, uint64_t b_bytes) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x < y + b_bytes && y < x + a_bytes;
}
}  // namespace bch
