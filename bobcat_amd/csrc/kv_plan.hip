// Plans of batches over the paged key/value cache: the host checks the
// sequences and their pages once a step, lays the work of the step's launches
// out, and copies it to the device, so that the kernels of every layer read a
// batch that is known to be in bounds.
#include <algorithm>
#include <cstdlib>
#include <cstring>
#include <memory>
#include <new>

#include "kernels.h"
#include "kv_cache.h"
#include "runtime.h"

namespace bch {

// Positions of a sequence and new tokens of a batch: a launch has fewer than 2^32
// threads, and kv_load and kv_store have 256 for every 16 positions and for
// every block that receives tokens.
constexpr uint32_t kKvMaxPositions = 1u << 27, kKvMaxTokens = 1u << 23;

static int check_shape(const char *kernel, const bch_kv_shape *s) {
  if (!s) return fail(BCH_ERR_ARGUMENT, "%s: no shape", kernel);
  if (s->format > BCH_KV_F8) return fail(BCH_ERR_UNSUPPORTED_FORMAT, "%s: no cache format %u", kernel, s->format);
  if (!s->n_kv_heads || s->n_kv_heads > 256 || (s->head_dim != 64 && s->head_dim != 128 && s->head_dim != 256))
    return fail(BCH_ERR_ATTENTION_LIMITS, "%s: 1 to 256 KV heads of 64, 128 or 256, got %u of %u", kernel,
                s->n_kv_heads, s->head_dim);
  if (!s->page_size || s->page_size % kKvBlock || s->page_size > kKvMaxPage || !s->n_pages)
    return fail(BCH_ERR_ARGUMENT, "%s: pages of 16 to %u positions, a multiple of 16, got %u pages of %u", kernel,
                kKvMaxPage, s->n_pages, s->page_size);
  return BCH_OK;
}

static int check_heads(const char *kernel, const bch_kv_shape *s, uint32_t n_heads) {
  if (!n_heads || n_heads % s->n_kv_heads || n_heads / s->n_kv_heads > kKvMaxGroup)
    return fail(BCH_ERR_ATTENTION_LIMITS, "%s: %u query heads over %u KV heads: groups of 1 to %u are wanted", kernel,
                n_heads, s->n_kv_heads, kKvMaxGroup);
  return BCH_OK;
}

static int check_batch(const char *kernel, const bch_kv_shape *s, uint32_t n_seqs, const uint32_t *n_past,
                       const uint32_t *n_new, const uint32_t *pages, uint64_t n_pages) {
  if (n_seqs && (!n_past || !n_new)) return fail(BCH_ERR_ARGUMENT, "%s: no lengths", kernel);
  if (n_pages && !pages) return fail(BCH_ERR_ARGUMENT, "%s: no pages", kernel);
  if (n_pages > 0x7fffffffu) return fail(BCH_ERR_ARGUMENT, "%s: more than 2^31 - 1 pages", kernel);
  uint64_t want = 0, tokens = 0;
  for (uint32_t i = 0; i < n_seqs; i++) {
    const uint64_t len = (uint64_t)n_past[i] + n_new[i];
    if (len > kKvMaxPositions)
      return fail(BCH_ERR_ARGUMENT, "%s: sequence %u has %llu positions", kernel, i, (unsigned long long)len);
    want += (len + s->page_size - 1) / s->page_size;
    tokens += n_new[i];
  }
  if (want != n_pages)
    return fail(BCH_ERR_ARGUMENT, "%s: the sequences need %llu pages, got %llu", kernel, (unsigned long long)want,
                (unsigned long long)n_pages);
  if (tokens > kKvMaxTokens) return fail(BCH_ERR_ARGUMENT, "%s: more than 2^23 new tokens", kernel);
  uint32_t last = 0;
  for (uint64_t i = 0; i < n_pages; i++) {
    if (pages[i] >= s->n_pages)
      return fail(BCH_ERR_OUT_OF_BOUNDS, "%s: page %u of a cache of %u pages", kernel, pages[i], s->n_pages);
    last = std::max(last, pages[i]);
  }
  // A page that receives tokens is named once in the whole batch: two
  // sequences (or two places of one) would overwrite each other's rows.  Pages
  // that are only read may be shared.  (calloc: of a large cache's counts only
  // those of the pages that are named are ever touched.)
  std::unique_ptr<uint8_t, decltype(&free)> counts(static_cast<uint8_t *>(calloc((size_t)last + 1, 1)), &free);
  if (!counts) throw std::bad_alloc();
  uint8_t *named = counts.get();
  for (uint64_t i = 0; i < n_pages; i++) named[pages[i]] = named[pages[i]] ? 2 : 1;
  uint64_t at = 0;
  for (uint32_t i = 0; i < n_seqs; i++) {
    const uint64_t len = (uint64_t)n_past[i] + n_new[i], n = (len + s->page_size - 1) / s->page_size;
    for (uint64_t p = n_past[i] / s->page_size; n_new[i] && p < n; p++)
      if (named[pages[at + p]] != 1)
        return fail(BCH_ERR_ARGUMENT, "%s: page %u receives tokens of sequence %u and is named twice", kernel,
                    pages[at + p], i);
    at += n;
  }
  return BCH_OK;
}

// The tokens' parents: each before its child, and trees of a size that masks are made for.
static bool is_chain(const uint32_t *parents, uint32_t n) {
  for (uint32_t i = 0; i < n; i++)
    if (parents[i] != (i ? i - 1 : BCH_NO_PARENT)) return false;
  return true;
}

static int check_trees(const char *kernel, uint32_t n_seqs, const uint32_t *n_new, const uint32_t *parents, uint64_t n_parents) {
  uint64_t tokens = 0;
  for (uint32_t i = 0; i < n_seqs; i++) tokens += n_new[i];
  if (n_parents != tokens)
    return fail(BCH_ERR_ARGUMENT, "%s: %llu parents for %llu new tokens", kernel, (unsigned long long)n_parents,
                (unsigned long long)tokens);
  if (tokens && !parents) return fail(BCH_ERR_ARGUMENT, "%s: no parents", kernel);
  for (uint32_t i = 0; i < n_seqs; parents += n_new[i++]) {
    if (is_chain(parents, n_new[i])) continue;
    if (n_new[i] > BCH_MAX_TREE)
      return fail(BCH_ERR_ARGUMENT, "%s: the tree of sequence %u has %u tokens, at most %u are wanted", kernel, i, n_new[i],
                  BCH_MAX_TREE);
    for (uint32_t t = 0; t < n_new[i]; t++)
      if (parents[t] != BCH_NO_PARENT && parents[t] >= t)
        return fail(BCH_ERR_ARGUMENT, "%s: token %u of sequence %u follows token %u", kernel, t, i, parents[t]);
  }
  return BCH_OK;
}

int kv_plan_ready(bch_ctx *ctx, const char *kernel, const bch_kv_plan *plan) {
  if (!plan) return fail(BCH_ERR_ARGUMENT, "%s: no plan", kernel);
  if (plan->ctx != ctx) return fail(BCH_ERR_FOREIGN_BUFFER, "%s: the plan belongs to another backend", kernel);
  if (!plan->ready) return fail(BCH_ERR_ARGUMENT, "%s: the plan has no batch", kernel);
  return BCH_OK;
}

int kv_plan_range(const char *kernel, const bch_kv_plan *plan, uint32_t first, uint32_t n, uint32_t *row, uint32_t *tokens) {
  if (first > plan->n_seqs || n > plan->n_seqs - first)
    return fail(BCH_ERR_ARGUMENT, "%s: sequences %u to %llu of %u", kernel, first, (unsigned long long)first + n, plan->n_seqs);
  auto at = [&](uint32_t seq) { return seq < plan->n_seqs ? plan->seqs[seq].row : plan->n_tokens; };
  *row = at(first);
  *tokens = at(first + n) - *row;
  return BCH_OK;
}

int kv_plan_cache(bch_ctx *ctx, const char *kernel, const bch_kv_plan *plan, bch_view cache, void **ptr) {
  BCH_TRY(kv_plan_ready(ctx, kernel, plan));
  BCH_TRY(check_view(ctx, kernel, cache, bch_kv_page_bytes(&plan->shape) * plan->shape.n_pages, ptr));
  if (reinterpret_cast<uintptr_t>(*ptr) % 16) return fail(BCH_ERR_ARGUMENT, "%s: the cache must be 16-byte aligned", kernel);
  return BCH_OK;
}

void kv_plan_use(const bch_ctx *ctx, const bch_kv_plan *plan) { plan->last_use = ctx->begun; }

int kv_plan_rows(bch_ctx *ctx, const char *kernel, const bch_kv_plan *plan, bch_view view, uint32_t width,
                 uint32_t stride, float **ptr) {
  if (stride < width || stride % 4)
    return fail(BCH_ERR_ARGUMENT, "%s: rows of %u floats %u apart: a multiple of 4 that holds them is wanted", kernel,
                width, stride);
  BCH_TRY(view_ptr(ctx, kernel, view, kv_rows_bytes(plan, width, stride), ptr));
  if (reinterpret_cast<uintptr_t>(*ptr) % 16) return fail(BCH_ERR_ARGUMENT, "%s: rows must be 16-byte aligned", kernel);
  return BCH_OK;
}

// Vectors of a batch, one behind the other in the plan's device memory.
struct Layout {
  std::vector<uint8_t> bytes;
  template <class T>
  uint64_t add(const T *data, uint64_t n) {
    const uint64_t at = (bytes.size() + 15) / 16 * 16;
    bytes.resize(at + n * sizeof(T));
    if (n) memcpy(bytes.data() + at, data, n * sizeof(T));
    return at;
  }
};

// The nodes and masks of a batch's trees; `rooted` as the plan's.
static void lay_trees(const std::vector<KvSeq> &seqs, const uint32_t *parents, std::vector<KvNode> &nodes,
                      std::vector<uint32_t> &masks, std::vector<uint8_t> &rooted) {
  for (const KvSeq &q : seqs) {
    const uint32_t *up = parents + q.row;
    const bool chain = is_chain(up, q.n_new);
    const uint32_t words = q.n_new && !chain ? kv_mask_words(q.past, q.n_new) : 0, skip = q.past % 32;
    KvNode *const of = nodes.data() + q.row;
    uint32_t roots = 0;
    std::vector<uint32_t> last(q.n_new, kKvNone);  // of a token's children so far
    for (uint32_t i = 0; i < q.n_new; i++) {
      const uint32_t a = up[i];
      of[i] = {a, kKvNone, kKvNone, a == BCH_NO_PARENT ? q.past : of[a].position + 1, words ? (uint32_t)masks.size() : kKvNone};
      if (a == BCH_NO_PARENT) {
        roots++;
      } else {
        (last[a] == kKvNone ? of[a].child : of[last[a]].sibling) = i;
        last[a] = i;
      }
      if (!words) continue;
      const size_t at = masks.size();
      masks.resize(at + words);
      if (a == BCH_NO_PARENT)
        masks[at] = (1u << skip) - 1;  // the past's keys of the first word
      else
        std::copy_n(masks.begin() + of[a].mask, words, masks.begin() + at);
      masks[at + (skip + i) / 32] |= 1u << (skip + i) % 32;
    }
    rooted.push_back(roots <= 1);
  }
}

static int plan_set(bch_kv_plan *plan, uint32_t n_seqs, const uint32_t *n_past, const uint32_t *n_new,
                    const uint32_t *pages, uint64_t n_pages, const uint32_t *parents) {
  const uint32_t page_blocks = plan->shape.page_size / kKvBlock;
  std::vector<KvSeq> seqs(n_seqs);
  std::vector<KvStoreItem> store;
  uint32_t row = 0, table = 0;
  for (uint32_t i = 0; i < n_seqs; i++) {
    const uint32_t end = n_past[i] + n_new[i];
    seqs[i] = {n_past[i], n_new[i], row, table};
    for (uint32_t p = n_past[i]; p < end;) {
      const uint32_t n = std::min(kKvBlock - p % kKvBlock, end - p);
      store.push_back({pages[table + p / kKvBlock / page_blocks], p, row + (p - n_past[i]), n});
      p += n;
    }
    row += n_new[i];
    table += (end + plan->shape.page_size - 1) / plan->shape.page_size;
  }
  // (Parents that make chains of all sequences are no trees.)
  std::vector<KvNode> nodes;
  std::vector<uint32_t> masks;
  std::vector<uint8_t> rooted;
  bool trees = false;
  for (uint32_t i = 0; parents && i < n_seqs; i++) trees |= !is_chain(parents + seqs[i].row, seqs[i].n_new);
  if (trees) {
    nodes.resize(row);
    lay_trees(seqs, parents, nodes, masks, rooted);
  }
  const KvSchedule work = kv_schedule(seqs, plan->n_heads / plan->shape.n_kv_heads, plan->shape.n_kv_heads,
                                      plan->shape.format, plan->shape.head_dim, plan->ctx->n_cus, plan->ctx->attn_partials ? kAttnPartialFloats : 0, trees);
  Layout all;
  const uint64_t at_seqs = all.add(seqs.data(), seqs.size());
  const uint64_t at_nodes = all.add(nodes.data(), nodes.size());
  const uint64_t at_masks = all.add(masks.data(), masks.size());
  const uint64_t at_pages = all.add(pages, n_pages);
  const uint64_t at_store = all.add(store.data(), store.size());
  const KvWork *const works[] = {&work.tiles8, &work.tiles16, &work.chunks};
  uint64_t at_items[3], at_starts[3];
  for (int i = 0; i < 3; i++) {
    at_items[i] = all.add(works[i]->items.data(), works[i]->items.size());
    at_starts[i] = all.add(works[i]->starts.data(), works[i]->starts.size());
  }
  const uint64_t at_join = all.add(work.join.data(), work.join.size());

  plan->ready = false;
  // Launches of a recording that was discarded have no ticket and may still
  // read the last batch.  (Where a later one was waited for they have run.)
  if (plan->last_use > plan->ctx->finished && hipStreamSynchronize(plan->ctx->stream) != hipSuccess)
    return fail(BCH_ERR_EXECUTION, "kv_plan_set: the stream failed");
  plan->last_use = 0;
  if (all.bytes.size() > plan->memory_bytes) {
    if (plan->memory) hipFree(plan->memory);
    plan->memory = nullptr;
    plan->memory_bytes = 0;
    const uint64_t room = all.bytes.size() + all.bytes.size() / 2;
    void *p = nullptr;
    if (hipMalloc(&p, room) != hipSuccess) {
      (void)hipGetLastError();
      return fail(BCH_ERR_ALLOCATION, "kv_plan_set: cannot allocate %llu bytes", (unsigned long long)room);
    }
    plan->memory = static_cast<uint8_t *>(p);
    plan->memory_bytes = room;
  }
  // Not on the context's stream, where the copy would wait for the steps of
  // other plans; done before this returns, so before any launch that reads it.
  if (!all.bytes.empty() &&
      (hipMemcpy(plan->memory, all.bytes.data(), all.bytes.size(), hipMemcpyHostToDevice) != hipSuccess ||
       hipStreamSynchronize(nullptr) != hipSuccess))
    return fail(BCH_ERR_EXECUTION, "kv_plan_set: host-to-device copy failed");
  plan->seqs.swap(seqs);
  plan->rooted.swap(rooted);
  plan->d_seqs = reinterpret_cast<const KvSeq *>(plan->memory + at_seqs);
  plan->d_nodes = trees ? reinterpret_cast<const KvNode *>(plan->memory + at_nodes) : nullptr;
  plan->d_masks = reinterpret_cast<const uint32_t *>(plan->memory + at_masks);
  plan->n_seqs = n_seqs;
  plan->n_tokens = row;
  plan->d_pages = reinterpret_cast<const uint32_t *>(plan->memory + at_pages);
  plan->d_store = reinterpret_cast<const KvStoreItem *>(plan->memory + at_store);
  plan->n_store = (uint32_t)store.size();
  bch_kv_plan::Work *const kept[] = {&plan->tiles8, &plan->tiles16, &plan->chunks};
  for (int i = 0; i < 3; i++)
    *kept[i] = {reinterpret_cast<const KvAttnItem *>(plan->memory + at_items[i]),
                works[i]->items.size() < works[i]->starts.size()
                    ? nullptr
                    : reinterpret_cast<const uint32_t *>(plan->memory + at_starts[i]),
                (uint32_t)works[i]->starts.size() - 1};
  plan->d_join = reinterpret_cast<const KvJoinItem *>(plan->memory + at_join);
  plan->tree_blocks = work.tree_blocks;
  plan->n_join = (uint32_t)work.join.size();
  plan->join_rows = plan->join_splits = 0;
  for (const KvJoinItem &j : work.join) {
    plan->join_rows = std::max(plan->join_rows, j.rows);
    plan->join_splits = std::max(plan->join_splits, j.splits);
  }
  plan->ready = true;
  return BCH_OK;
}

}  // namespace bch

using namespace bch;

extern "C" {

uint64_t bch_kv_page_bytes(const bch_kv_shape *shape) {
  if (check_shape("kv_page_bytes", shape) != BCH_OK) return 0;
  return (uint64_t)shape->n_kv_heads * (shape->page_size / kKvBlock) * kv_block_bytes(shape->format, shape->head_dim);
}

static int plan_check(const bch_kv_shape *shape, uint32_t n_heads, uint32_t n_seqs, const uint32_t *n_past,
                      const uint32_t *n_new, const uint32_t *pages, uint64_t n_pages, bool trees, const uint32_t *parents,
                      uint64_t n_parents) {
  BCH_TRY(check_shape("kv_plan", shape));
  BCH_TRY(check_heads("kv_plan", shape, n_heads));
  try {
    BCH_TRY(check_batch("kv_plan", shape, n_seqs, n_past, n_new, pages, n_pages));
  } catch (const std::bad_alloc &) {
    return fail(BCH_ERR_ALLOCATION, "kv_plan: out of host memory");
  }
  return trees ? check_trees("kv_plan", n_seqs, n_new, parents, n_parents) : BCH_OK;
}

int bch_kv_plan_check(const bch_kv_shape *shape, uint32_t n_heads, uint32_t n_seqs, const uint32_t *n_past,
                      const uint32_t *n_new, const uint32_t *pages, uint64_t n_pages) {
  return plan_check(shape, n_heads, n_seqs, n_past, n_new, pages, n_pages, false, nullptr, 0);
}

int bch_kv_plan_check_trees(const bch_kv_shape *shape, uint32_t n_heads, uint32_t n_seqs, const uint32_t *n_past,
                            const uint32_t *n_new, const uint32_t *pages, uint64_t n_pages, const uint32_t *parents,
                            uint64_t n_parents) {
  return plan_check(shape, n_heads, n_seqs, n_past, n_new, pages, n_pages, true, parents, n_parents);
}

int bch_kv_plan_new(bch_ctx *ctx, const bch_kv_shape *shape, uint32_t n_heads, bch_kv_plan **out) {
  if (!out) return fail(BCH_ERR_ARGUMENT, "kv_plan: nowhere to store the plan");
  *out = nullptr;
  BCH_TRY(check_shape("kv_plan", shape));
  BCH_TRY(check_heads("kv_plan", shape, n_heads));
  if (!ctx) return fail(BCH_ERR_ARGUMENT, "kv_plan: no backend");
  auto *plan = new (std::nothrow) bch_kv_plan;
  if (!plan) return fail(BCH_ERR_ALLOCATION, "kv_plan: out of host memory");
  plan->ctx = ctx;
  plan->shape = *shape;
  plan->n_heads = n_heads;
  *out = plan;
  return BCH_OK;
}

void bch_kv_plan_free(bch_kv_plan *plan) {
  if (!plan) return;
  if (plan->memory) {
    hipStreamSynchronize(plan->ctx->stream);
    hipFree(plan->memory);
  }
  delete plan;
}

static int plan_take(bch_kv_plan *plan, uint32_t n_seqs, const uint32_t *n_past, const uint32_t *n_new,
                     const uint32_t *pages, uint64_t n_pages, bool trees, const uint32_t *parents, uint64_t n_parents) {
  if (!plan) return fail(BCH_ERR_ARGUMENT, "kv_plan_set: no plan");
  // In the open recording, or in one that has not been waited for.
  const bch_ctx *ctx = plan->ctx;
  bool busy = ctx->recording && plan->last_use == ctx->begun;
  for (const bch_ctx::Pending &p : ctx->pending) busy |= plan->last_use == p.recording;
  if (busy)
    return fail(BCH_ERR_BUSY, "kv_plan_set: the batch cannot change while work that uses it is in flight");
  BCH_TRY(plan_check(&plan->shape, plan->n_heads, n_seqs, n_past, n_new, pages, n_pages, trees, parents, n_parents));
  try {
    return plan_set(plan, n_seqs, n_past, n_new, pages, n_pages, trees ? parents : nullptr);
  } catch (const std::bad_alloc &) {
    return fail(BCH_ERR_ALLOCATION, "kv_plan_set: out of host memory");
  }
}

int bch_kv_plan_set(bch_kv_plan *plan, uint32_t n_seqs, const uint32_t *n_past, const uint32_t *n_new,
                    const uint32_t *pages, uint64_t n_pages) {
  return plan_take(plan, n_seqs, n_past, n_new, pages, n_pages, false, nullptr, 0);
}

int bch_kv_plan_set_trees(bch_kv_plan *plan, uint32_t n_seqs, const uint32_t *n_past, const uint32_t *n_new,
                          const uint32_t *pages, uint64_t n_pages, const uint32_t *parents, uint64_t n_parents) {
  return plan_take(plan, n_seqs, n_past, n_new, pages, n_pages, true, parents, n_parents);
}

}  // extern "C"
