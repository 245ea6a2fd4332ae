// Attention of a batch's new tokens over the paged cache: the join of split keys,
// the work of a batch, and the entry point.  (The tiles' kernels: attn_paged.h.)
#include <algorithm>
#include <cmath>
#include <numeric>

#include "attn_paged.h"

namespace bch {

// The rows of tiles whose keys were split, from the splits' records.  HD / 4
// threads read a record; `parts` (a power of two) such groups have every
// parts-th of a row's records each and meet in LDS.  Bound by latency (the item,
// then its records): 4.3 us for rows of up to 16 pieces.  Eight records in flight
// each, three where there are no more: 50 wide and some narrow tiles of heads of
// 128, 58 MB of records, 28 us instead of 32.
template <uint32_t HD>
__global__ __launch_bounds__(256) void k_attn_join(const KvJoinItem *__restrict__ items, uint32_t n_kv, uint32_t group,
                                                   uint32_t parts, AttnOut to) {
  constexpr uint32_t WIDE = HD / 4, GROUPS = 256 / WIDE;
  __shared__ float4 acc_s[GROUPS][WIDE];
  __shared__ float2 ml_s[GROUPS];
  const KvJoinItem it = items[blockIdx.x];
  const uint32_t kv = blockIdx.y, lane = threadIdx.x % WIDE, mine = threadIdx.x / WIDE, part = mine % parts, d = 4 * lane;
  const uint32_t row = blockIdx.z * (GROUPS / parts) + mine / parts;
  if (blockIdx.z * (GROUPS / parts) >= it.rows) return;
  const uint64_t apart = (uint64_t)n_kv * it.rows * (HD + 4);
  const float *p = to.partials + ((uint64_t)it.part + kv * it.rows + min(row, it.rows - 1)) * (HD + 4);
  float top = -INFINITY, sum = 0.f;
  float4 acc = {0.f, 0.f, 0.f, 0.f};
  // The weight of a reference m under another that is no smaller.
  auto weight = [](float m, float under) { return m == under ? 1.f : __builtin_amdgcn_exp2f(m - under); };
  auto add = [&](float f, float4 x, float l) {
    acc.x = fmaf(x.x, f, acc.x), acc.y = fmaf(x.y, f, acc.y), acc.z = fmaf(x.z, f, acc.z), acc.w = fmaf(x.w, f, acc.w);
    sum = fmaf(l, f, sum);
  };
  auto take = [&](auto in_flight) __attribute__((always_inline)) {
    constexpr uint32_t N = decltype(in_flight)::value;
    for (uint32_t s0 = part; s0 < it.splits; s0 += N * parts) {
      float2 ml[N];
      float4 x[N];
#pragma unroll
      for (uint32_t j = 0; j < N; j++) {
        const float *r = p + min(s0 + j * parts, it.splits - 1) * apart;
        ml[j] = *reinterpret_cast<const float2 *>(r + HD);
        x[j] = *reinterpret_cast<const float4 *>(r + d);
      }
      float next = top;
#pragma unroll
      for (uint32_t j = 0; j < N; j++) next = fmaxf(next, ml[j].x);
      const float f0 = weight(top, next);
      top = next;
      sum *= f0;
      acc.x *= f0, acc.y *= f0, acc.z *= f0, acc.w *= f0;
#pragma unroll
      for (uint32_t j = 0; j < N; j++) {
        if (s0 + j * parts >= it.splits) break;
        add(weight(ml[j].x, top), x[j], ml[j].y);
      }
    }
  };
  if (it.splits <= 3 * parts)
    take(std::integral_constant<uint32_t, 3>{});
  else
    take(std::integral_constant<uint32_t, 8>{});
  if (parts > 1) {
    acc_s[mine][lane] = acc;
    if (lane == 0) ml_s[mine] = {top, sum};
    __syncthreads();
    if (part) return;
    float all = top;
    for (uint32_t j = 1; j < parts; j++) all = fmaxf(all, ml_s[mine + j].x);
    const float f0 = weight(top, all);
    acc.x *= f0, acc.y *= f0, acc.z *= f0, acc.w *= f0;
    sum *= f0;
    for (uint32_t j = 1; j < parts; j++) add(weight(ml_s[mine + j].x, all), acc_s[mine + j][lane], ml_s[mine + j].y);
    top = all;
  }
  if (row >= it.rows) return;
  const uint32_t at = it.first + row;
  put_row<HD>(to, ~0u, 0, it.row + at / group, kv * group + at % group, d, acc, top, sum);
}

// --- the work of a batch ----------------------------------------------------------

// Tiles whose rows are dealt out, with their keys in steps of 32.
struct Tile {
  KvAttnItem it;
  uint32_t steps;
};

// Deals the tiles' steps to workgroups, at most `most` for each KV head so that
// all run at once, in one of two ways.  Evenly: a tile makes pieces of about one
// length, `least` steps or more, a workgroup each.  Or in equal shares: a tile is
// cut where a workgroup's share ends, which then goes on with the next tile, and
// all workgroups end together.  A piece counts `start` steps besides its own
// (its queries, the first keys' way, its results); the way whose longest
// workgroup is shorter is taken.  (Heads of 64, 12 sequences of 96 rows: 31 us
// evenly, 34 in shares; of 128, 56 tiles of 200 to 500 steps for 64 workgroups:
// 834 and 800.)  With `whole` no tile is cut.
struct Dealer {
  const std::vector<Tile> &tiles;
  uint64_t most;
  uint32_t least;
  bool whole;
  uint64_t start;
  uint32_t granule;

  // Pieces of a tile at an even length of n steps.
  uint32_t pieces(const Tile &t, uint32_t n) const { return whole ? 1u : std::max((t.steps + n / 2) / n, 1u); }

  // put(tile, lo, hi) for every piece, next() between workgroups.
  template <class Put, class Next>
  void evenly(uint32_t n, Put &&put, Next &&next) const {
    for (const Tile &t : tiles) {
      const uint32_t parts = pieces(t, n), units = (t.steps + granule - 1) / granule;
      for (uint32_t i = 0; i < parts; i++) {
        put(t, (uint32_t)((uint64_t)units * i / parts) * granule,
            std::min((uint32_t)((uint64_t)units * (i + 1) / parts) * granule, t.steps));
        next();
      }
    }
  }
  template <class Put, class Next>
  void shares(uint64_t share, Put &&put, Next &&next) const {
    uint64_t room = share;
    for (const Tile &t : tiles)
      for (uint32_t at = 0; at < t.steps;) {
        const uint32_t left = t.steps - at;
        if (room < share && room < (whole ? left : std::min(left, least)) + start) {  // no room for a piece
          next();
          room = share;
        }
        uint32_t take = left;
        if (!whole && room < left + start && left >= 2 * least)
          take = std::max(std::min(std::max((uint32_t)(room - start), least), left - least) / granule * granule, granule);
        put(t, at, at + take);
        at += take;
        room -= std::min<uint64_t>(room, take + start);
      }
  }
};

// Workgroups go to the eight XCDs in turn, so those of a KV head to
// 8 / gcd(8, n_kv) of them.  Puts the pieces of a sequence's tiles that read the
// same keys on one XCD, whose L2 then has them for all but the first.
static void keep_together(std::vector<KvAttnItem> &items, uint32_t n_kv) {
  const uint32_t xcds = 8 / std::gcd(8u, n_kv);
  if (xcds == 1) return;
  struct Piece {
    uint32_t row, number;
    KvAttnItem it;
  };
  std::vector<Piece> pieces;
  pieces.reserve(items.size());
  for (const KvAttnItem &it : items) {
    const bool same = !pieces.empty() && pieces.back().row == it.row && pieces.back().it.first == it.first;
    pieces.push_back({it.row, same ? pieces.back().number + 1 : 0, it});
  }
  auto before = [](const Piece &a, const Piece &b) { return a.row != b.row ? a.row < b.row : a.number < b.number; };
  std::stable_sort(pieces.begin(), pieces.end(), before);
  std::vector<KvAttnItem> of[8];
  uint32_t to = 0;
  for (size_t i = 0; i < pieces.size(); i++) {
    if (!i || before(pieces[i - 1], pieces[i])) {
      for (uint32_t x = to = 0; x < xcds; x++)
        if (of[x].size() < of[to].size()) to = x;
    }
    of[to].push_back(pieces[i].it);
  }
  items.clear();
  for (size_t i = 0; items.size() < pieces.size(); i++)
    for (uint32_t x = 0; x < xcds; x++)
      if (i < of[x].size()) items.push_back(of[x][i]);
}

static void deal(KvSchedule &w, KvWork &work, const std::vector<Tile> &tiles, uint64_t most, uint32_t least, bool whole,
                 uint64_t start, uint32_t n_kv, uint32_t granule, uint64_t records) {
  work.starts.push_back(0);
  if (tiles.empty()) return;
  Dealer d{tiles, std::max<uint64_t>(most, 1), least, whole, start, granule};
  uint64_t total = 0, room = w.records;
  uint32_t longest = 1;
  for (const Tile &t : tiles) {
    total += t.steps + start;
    longest = std::max(longest, t.steps);
  }
  // The smallest length and share that make no more than `most` workgroups.
  auto smallest = [](uint64_t lo, uint64_t hi, auto &&fits) {
    while (lo < hi) {
      const uint64_t mid = lo + (hi - lo) / 2;
      if (fits(mid)) hi = mid; else lo = mid + 1;
    }
    return lo;
  };
  auto none = [](const Tile &, uint32_t, uint32_t) {};
  const uint32_t even = (uint32_t)smallest(least, 2ull * std::max(longest, least), [&](uint64_t n) {
    uint64_t sum = 0;
    for (const Tile &t : tiles) sum += d.pieces(t, (uint32_t)n);
    return sum <= d.most;
  });
  uint64_t even_groups = 0, even_end = 0;
  for (const Tile &t : tiles) {
    even_groups += d.pieces(t, even);
    even_end = std::max<uint64_t>(even_end, t.steps / d.pieces(t, even) + start);
  }
  const uint64_t share = smallest(std::max<uint64_t>(total / d.most, least + start), total + 1, [&](uint64_t n) {
    uint64_t groups = 1;
    d.shares(n, none, [&] { groups++; });
    return groups <= d.most;
  });
  const bool evenly = even_groups <= d.most && even_end <= share;
  // Partial results of more pieces than have room: no tile is cut.
  auto need = [&](const Tile &t, uint32_t lo, uint32_t hi) {
    if (hi - lo < t.steps) room += (uint64_t)n_kv * t.it.rows;
  };
  if (evenly)
    d.evenly(even, need, [] {});
  else
    d.shares(share, need, [] {});
  if (room > records) d.whole = true;

  const Tile *open = nullptr;  // the tile that the last piece was of
  auto put = [&](const Tile &t, uint32_t lo, uint32_t hi) {
    KvAttnItem it = t.it;
    it.lo = lo;
    it.hi = hi;
    if (hi - lo < t.steps) {
      if (open != &t) w.join.push_back({it.row, it.first, it.rows, 0, (uint32_t)w.records});
      w.join.back().splits++;
      it.part = (uint32_t)w.records;
      w.records += (uint64_t)n_kv * it.rows;
    }
    open = &t;
    work.items.push_back(it);
  };
  auto next = [&] { work.starts.push_back((uint32_t)work.items.size()); };
  if (evenly)
    d.evenly(even, put, next);
  else
    d.shares(share, put, next);
  if (work.starts.back() != work.items.size()) next();
}

// Which tiles a batch with trees takes: wide ones, or narrow ones of up to `blocks` times 16
// rows.  Narrow tiles cost about the same for every block and step of 32 keys once
// there is work for all waves; a wide one as much as 6.3 blocks in the 8-bit formats,
// where a narrow tile widens the keys for itself, and 5 in f16, or 3 from 128 MB of keys
// and values on, which the narrow tiles of a tree bring one after the other.  (32 sequences of up to 6,000 keys, eight KV heads of 128, up to 48, 64, 128
// and 192 rows: int8 82, 106, 177, 213 us narrow and 132, 142, 174, 216 wide; f16 109, 147, 256,
// 359 and 151, 136, 184, 272.)  Below 16 steps of a block for each wave the time is latency, and tiles of
// one block share it among more waves (one sequence of 600 keys and 32 rows, heads of 64: 8.2
// us, in tiles of two 11.3, wide 20.6; twelve of up to 2,500 keys and 96 rows 21, 24 and 36).  Not so in f16 from 96 MB
// on: five sequences of up to 12,868 keys and 48
// rows, heads of 128, 70 us in tiles of one block and 54 by the rule for large batches; eight of up to 6,000 and 64
// rows 55 and 48; but three of up to 16,000, 90 MB, 32 and 46, and in int8 20 of up to 6,000 43 and 50.  Three
// blocks beat two only where there is much more (12 of 256 rows: 52 us and 45; 32 of 96 rows and 6,000 keys 73
// and 75).  Both edges are measured ones, not a cache's size (the last one has 256 MB): over 81 f16 batches of 47 to 283 MB
// the rule is within 12% of the best choice but for four, 17 to 25% (profiles/tree_tiles_choice.txt).
// A prompt in the batch counts with the trees.  It needs the wide kernel in any case, and trees in narrow tiles are
// a launch more: beside 1,024 or 2,048 tokens the rule takes wide tiles for them, which cost up to 5% more than narrow
// ones (16 trees of 8 tokens, int8, 86.8 us and 82.6) and up to 17% less; beside 256 tokens it mostly takes narrow ones,
// up to 38% more than wide ones (16 of 8, f16, heads of 64, 42 us and 30.5).  In none of 90 such batches is one plan
// more than 5% behind two, the prompt's and the trees'.
struct TreeTiles {
  bool wide;
  uint32_t blocks;
};
static TreeTiles tree_tiles(const std::vector<KvSeq> &seqs, uint32_t group, uint32_t n_kv, uint32_t format,
                            uint32_t head_dim, uint32_t n_cus) {
  uint64_t block_steps = 0, wide_steps = 0, keys = 0, most = 1;
  for (const KvSeq &q : seqs) {
    const uint64_t rows = (uint64_t)q.n_new * group, steps = (q.past + q.n_new + 31) / 32;
    most = std::max(most, (rows + 15) / 16);
    block_steps += (rows + 15) / 16 * steps;
    wide_steps += (rows + kChunkRows - 1) / kChunkRows * steps;
    keys += q.past + q.n_new;
  }
  const uint64_t waves = 4ull * n_cus * tree_tile_groups(format, head_dim, 1), work = block_steps * n_kv;
  const uint64_t bytes = keys * n_kv * kv_block_bytes(format, head_dim) / kKvBlock;
  const bool shared = format != BCH_KV_F16 || bytes <= (96ull << 20);
  if (most == 1 || (work <= 16 * waves && shared)) return {false, 1};
  const double ratio = format != BCH_KV_F16 ? 6.3 : bytes <= (128ull << 20) ? 5.0 : 3.0;
  if (ratio * wide_steps < block_steps) return {true, 1};
  return {false, std::min(work <= 32 * waves ? 2u : 3u, tree_tile_rows(format, head_dim) / 16)};
}

KvSchedule kv_schedule(const std::vector<KvSeq> &seqs, uint32_t group, uint32_t n_kv, uint32_t format, uint32_t head_dim,
                       uint32_t n_cus, uint64_t partial_floats, bool trees) {
  KvSchedule w;
  const uint64_t records = std::min<uint64_t>(partial_floats / (head_dim + 4), 0xfffffffeu);
  if (!n_cus) n_cus = 256;
  // Which tiles.  Narrow ones read the keys again for every 16 rows but share
  // them out among the waves; in a wide one's the waves share the keys, and idle
  // where there are no rows for them.  Twelve sequences of about 2,000 keys, 20,
  // 64, 96 and 128 rows: 17, 27, 28 and 44 us in narrow tiles, 26, 28, 31 and 36
  // in wide ones (heads of 64; of 128: 20, 31, 48, 64 and 36, 36, 49, 58; of 256:
  // 18, 30, 41, 48 and 44, 38, 48, 51).  One sequence of 128 rows and 1,000 keys:
  // 12 and 20.  Where some sequence needs wide tiles, only those of up to 32 rows
  // stay narrow, since a second launch costs more than the rows that idle.
  constexpr uint64_t kSmallBatch = 1u << 20;  // narrow tiles x steps x KV heads x head_dim
  uint64_t narrow_work = 0;
  bool wide = false, large = false;
  for (const KvSeq &q : seqs) {
    const uint64_t rows = (uint64_t)q.n_new * group;
    wide |= rows > kChunkRows;
    large |= rows > 96;
    if (rows > 16 && rows <= kChunkRows) narrow_work += (rows + 15) / 16 * ((q.past + q.n_new + 31) / 32) * n_kv * head_dim;
  }
  const TreeTiles tree = trees ? tree_tiles(seqs, group, n_kv, format, head_dim, n_cus) : TreeTiles{};
  w.tree_blocks = tree.blocks;
  // (Beside trees in wide tiles what one block holds stays narrow, beside others a prompt is wide.)
  const uint32_t few_rows = trees ? (tree.wide ? 16 : 4 * kChunkRows)
                                  : wide || (large && narrow_work > kSmallBatch) ? 32 : kChunkRows;
  std::vector<Tile> narrow, tokens, chunks;
  uint32_t longest = 0;
  uint64_t narrow_steps = 0, token_steps = 0;
  for (const KvSeq &q : seqs) {
    const uint32_t rows = q.n_new * group;
    const bool few = rows <= few_rows;
    // (A tree's in equal tiles of whole blocks.)
    const uint32_t most = trees ? 16 * tree.blocks : 16, tiles = (rows + most - 1) / most;
    const uint32_t narrow_rows = !trees || !tiles ? 16 : ((rows + 15) / 16 + tiles - 1) / tiles * 16;
    for (uint32_t first = 0; first < rows; first += few ? narrow_rows : kChunkRows) {
      const uint32_t n = std::min(few ? narrow_rows : kChunkRows, rows - first), keys = q.past + (first + n - 1) / group + 1;
      const Tile t{{q.table, q.past, q.row, first, n, 0, 0, ~0u}, (keys + 31) / 32};
      (!few ? chunks : n <= 8 && !trees ? narrow : tokens).push_back(t);
      if (few) {
        longest = std::max(longest, t.steps);
        (n <= 8 ? narrow_steps : token_steps) += t.steps;
      }
    }
  }
  // A few tiles of 8 rows join those of 16 in one launch.
  if (narrow_steps <= token_steps) {
    tokens.insert(tokens.end(), narrow.begin(), narrow.end());
    narrow.clear();
  }
  // Narrow tiles: pieces of eight steps (two a wave) are as short as pays, and
  // a join (about 2.5 us) pays from 24 steps on with heads of 64, 19 of 128, 16
  // of 256 (300 keys of 64: 5.6 us whole, 7.6 cut; 2,000: 14.2 and 9.0).
  const uint32_t unsplit = 14 + 640 / head_dim;
  // What the registers let run at once; of heads of 256 one a CU: twelve
  // sequences of five drafts in int8 19.6 us, with two 23.4, in e4m3 18.1 and 23.0.
  // (Where a sequence has one tile it goes both ways: single tokens of 64
  // sequences of 4,000 int8 keys, two KV heads, 29.8 and 27.9; of eight, eight KV
  // heads, 24.4 and 22.2, in e4m3 16.2 and 17.9; of one with 32,000 keys 29.4 and
  // 30.6.)
  const uint32_t at_once = trees ? tree_tile_groups(format, head_dim, tree.blocks) : head_dim == 256 ? 1 : token_groups(format, head_dim);
  const uint64_t few_groups = (uint64_t)n_cus * at_once / n_kv;
  deal(w, w.tiles8, narrow, few_groups, 8, longest <= unsplit, 4, n_kv, 1, records);
  deal(w, w.tiles16, tokens, few_groups, 8, longest <= unsplit, 4, n_kv, 1, records);
  // Where a workgroup has one item, the order is free.  (Heads of 256, 12 sequences
  // of 20 rows and 4,096 keys: 18.1 us instead of 20.4 in e4m3, 23.4 instead of
  // 26.2 in f16, of 64 rows and 2,000 keys 18.7 instead of 19.8; single tokens,
  // whose tiles share no keys, the same either way.  Smaller heads take fewer bytes
  // a CU at a time and gain nothing: of 128, 20 rows, 15.5 instead of 15.0, of 64
  // 12.3 and 12.3.)
  if (head_dim == 256)
    for (KvWork *work : {&w.tiles8, &w.tiles16})
      if (work->items.size() < work->starts.size()) keep_together(work->items, n_kv);
  const uint32_t keys = chunk_keys(format, head_dim);
  // Wide tiles: four trips of the loop at least.  What starting one costs showed
  // in prompts without a past, 2,048 tokens in 64 tiles of 1 to 64 steps (heads of
  // 128): 156 us counted as 4 steps, 114 as 10.
  deal(w, w.chunks, chunks, (uint64_t)n_cus * chunk_groups(format, head_dim) / n_kv, keys / 8, false, 10, n_kv,
       keys / 32, records);
  return w;
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
    kv_plan_use(ctx, plan);
    const uint32_t n_kv = s.n_kv_heads, group = plan->n_heads / n_kv;
    const AttnOut to{op, out_stride, ctx->attn_partials};
    const AttnCall call{st, plan, plan->geometry(cp), qp, q_stride, group, to,
                        (float)(1.44269504088896340736 / std::sqrt((double)s.head_dim))};
    if (plan->d_nodes) launch_tree_tiles(call);
    kv_dispatch(s.format, s.head_dim, [&](auto format, auto hd) {
      constexpr uint32_t F = decltype(format)::value, HD = decltype(hd)::value;
      const bch_kv_plan::Work &c = plan->chunks, &t16 = plan->tiles16, &t8 = plan->tiles8;
      if (!plan->d_nodes) {
        if (c.groups)
          k_attn_chunk<F, HD, false><<<c.groups * n_kv, 256, 0, st>>>(call.geo, c.items, c.starts, qp, q_stride, to, group,
                                                                      call.c2, {});
        if (t16.groups)
          k_attn_tokens<F, HD, 16><<<t16.groups * n_kv, 256, 0, st>>>(call.geo, t16.items, t16.starts, qp, q_stride, to, group, call.c2);
        if (t8.groups)
          k_attn_tokens<F, HD, 8><<<t8.groups * n_kv, 256, 0, st>>>(call.geo, t8.items, t8.starts, qp, q_stride, to, group, call.c2);
      }
      if (plan->n_join) {
        // Up to eight records each in one round of loads.
        constexpr uint32_t kGroups = 1024 / HD;
        uint32_t parts = 1;
        while (parts < kGroups && parts * 8 < plan->join_splits) parts *= 2;
        k_attn_join<HD><<<dim3(plan->n_join, n_kv, div_ceil(plan->join_rows * parts, kGroups)), 256, 0, st>>>(
            plan->d_join, n_kv, group, parts, to);
      }
    });
  });
}
