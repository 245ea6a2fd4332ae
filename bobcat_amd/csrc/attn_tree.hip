// Attention over the paged cache where a batch's new tokens are trees.
//
// The rows are packed as elsewhere (attn_paged.h), a few dozen of them for a
// sequence: more than one 16-column operand holds, fewer than the waves of a wide
// tile want.  k_attn_tree takes up to 16·NB of them at a time: a wave brings 32
// keys of its own into registers, widens them once, and multiplies them with
// each of the NB blocks of 16 rows; the waves of a workgroup, and the pieces of
// a tile, have other keys and are joined.  Trees of more rows go to the wide tiles.
//
// What bounds it is the vector work beside the MFMAs: per 32 keys 40 instructions
// to widen the 8-bit keys, 40 for the values, and per block of 16 rows about 75 for
// the softmax, half of them for 8 exponentials; the MFMAs of a block take 64 issue
// slots.  32 trees of 12 to 24 tokens over 1,024 to 8,192 int8 positions, 8 KV heads of
// 64, 32 heads: 97-105 us and the join 4.6 (the cache's bytes at a copy's rate 34, both parts'
// products at a library's rate 40); 12 of 6 to 12 over up to 4,096, e4m3, two KV heads of 256,
// 20.6 and 4.4; one of 8 tokens over 600 8.0, by latency.  Wide tiles: 8 trees of 32 to 64
// tokens over up to 12,000 f16 positions, 8 KV heads of 128, 142-148 and 11.
#include <algorithm>

#include "attn_paged.h"

namespace bch {

// Blocks of 16 rows of a tile at most, and workgroups of a CU of a kernel for up to `most`: what
// the registers hold of queries and outputs (2·hd / 4 a block) beside the keys on their way.  16
// sequences of up to 8,192 positions (the GPU's time, the join's with it), int8, heads of 64 with
// 96 rows: 62 us, one workgroup a CU 75, four blocks 63; of 128: 90, three blocks 239 (it spills),
// one block 104; of 256, two KV heads: 70, two blocks 76.  f16, heads of 128, 32 rows of 32
// sequences of up to 6,000: two blocks with one workgroup a CU 99, one block with two 120;
// but 12 of up to 2,500, 48 rows, 39 and 30: so there is a kernel for each.  f16, heads of 256, 64 rows,
// one workgroup a CU 76, two 108 (it spills).  (In 8 bits 7 to 14 registers are spilled with heads of 128, 14 to 17 with
// heads of 256, where an item begins; the loop of whole steps reloads none, that of masked ones 7 of heads of 256.)
constexpr uint32_t tree_blocks(uint32_t format, uint32_t hd) {
  return hd == 64 ? (format == BCH_KV_F16 ? 2 : 3) : hd == 128 ? 2 : 1;
}
constexpr uint32_t tree_groups(uint32_t format, uint32_t hd, uint32_t most) {
  return format == BCH_KV_F16 && (hd == 256 || (hd == 128 && most > 1)) ? 1 : 2;
}
// The kernel of a batch whose tiles have up to `blocks`.
constexpr uint32_t tree_most(uint32_t format, uint32_t hd, uint32_t blocks) {
  const uint32_t most = tree_blocks(format, hd);
  return blocks > 1 || tree_groups(format, hd, 1) == tree_groups(format, hd, most) ? most : 1;
}

uint32_t tree_tile_rows(uint32_t format, uint32_t hd) { return 16 * tree_blocks(format, hd); }
uint32_t tree_tile_groups(uint32_t format, uint32_t hd, uint32_t blocks) {
  return tree_groups(format, hd, tree_most(format, hd, blocks));
}

template <uint32_t FORMAT, uint32_t HD, uint32_t MOST>
__global__ __launch_bounds__(256, tree_groups(FORMAT, HD, MOST)) void k_attn_tree(
    KvGeometry g, const KvAttnItem *__restrict__ items, const uint32_t *__restrict__ starts, const float *__restrict__ q,
    uint32_t q_stride, AttnOut to, uint32_t group, float c2, AttnTrees trees) {
  constexpr bool QUANT = FORMAT != BCH_KV_F16;
  constexpr uint32_t SIZE = kv_elem_bytes(FORMAT), BYTES = kv_block_bytes(FORMAT, HD), PART = kKvBlock * HD * SIZE;
  constexpr uint32_t NL = PART / 1024, KS = HD / 32, OB = HD / 16, M = 4 / SIZE;
  __shared__ __align__(16) float o_s[4][16][HD];
  __shared__ float m_s[4][16], l_s[4][16];
  const uint32_t kv = blockIdx.x % g.n_kv, share = blockIdx.x / g.n_kv, end = starts ? starts[share + 1] : share + 1;
  // A tile of NB blocks of rows.  (Blocks that a tile lacks are left out by code of its
  // own for each number: conditions around each block's instructions kept them apart.)
  auto tile = [&](const KvAttnItem &it, auto blocks) __attribute__((always_inline)) {
    constexpr uint32_t NB = decltype(blocks)::value;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
    const uint32_t col = lane % 16, quad = lane / 16;
    const uint32_t n_keys = it.past + (it.first + it.rows - 1) / group + 1, last = (n_keys - 1) / kKvBlock;
    // Keys that every row of the tile sees.
    const bool tree = trees.nodes[it.row].mask != kKvNone;
    const int whole = tree ? it.past : it.past + it.first / group + 1;

    struct Raw {
      au4_t x[2][NL];
      float4 s[2];
    } kr, vr;
    // (Past the end: the last block, masked.)  A step's page numbers are brought a step before its
    // keys, so that these wait for nothing.
    struct Pages {
      uint32_t x[2];
    };
    auto pages_of = [&](uint32_t step) __attribute__((always_inline)) {
      return Pages{{g.page(it.table, min(2 * step, last)), g.page(it.table, min(2 * step + 1, last))}};
    };
    auto load = [&](Raw &raw, const Pages &pages, uint32_t step, uint32_t part) __attribute__((always_inline)) {
#pragma unroll
      for (int t = 0; t < 2; t++) {
        const uint8_t *p = g.block<BYTES>(pages.x[t], min(2 * step + t, last), kv);
#pragma unroll
        for (uint32_t c = 0; c < NL; c++)
          raw.x[t][c] = *reinterpret_cast<const au4_t *>(p + part * PART + 1024 * c + 16 * lane);
        if constexpr (QUANT) raw.s[t] = *reinterpret_cast<const float4 *>(p + 2 * PART + 64 * part + 16 * quad);
      }
    };
    uint32_t step = it.lo + wave;
    auto after = [&](uint32_t step) { return min(step + 4, it.hi - 1); };
    Pages pages;  // of the next step
    if (step < it.hi) {
      const Pages now = pages_of(step);
      pages = pages_of(after(step));
      load(kr, now, step, 0);
      load(vr, now, step, 1);
    }

    // The rows' elements as the keys' operand has them (k_attn_tokens), and where a row's mask
    // has key 0 (of a chain: its position).
    ah8_t qh[NB][KS], ql[NB][KS];
    float back[NB], m[NB], l[NB], lazy[NB], x[NB][KS][8];
    uint32_t sees_at[NB];
#pragma unroll
    for (uint32_t n = 0; n < NB; n++) {
      const uint32_t packed = it.first + min(16 * n + col, it.rows - 1), token = packed / group, head = kv * group + packed % group;
      sees_at[n] = tree ? trees.nodes[it.row + token].mask - it.past / 32 : it.past + token;  // (of key 0: it may wrap)
      m[n] = l[n] = 0.f, lazy[n] = kUnset;
      const float *qr = q + (uint64_t)(it.row + token) * q_stride + (uint64_t)head * HD;
#pragma unroll
      for (uint32_t s = 0; s < KS; s++) {
        const uint32_t e = QUANT ? 64 * (s / 2) + 16 * quad + 8 * (s % 2) : 32 * s + 8 * quad;
        const float4 a = *reinterpret_cast<const float4 *>(qr + e), b = *reinterpret_cast<const float4 *>(qr + e + 4);
        x[n][s][0] = a.x, x[n][s][1] = a.y, x[n][s][2] = a.z, x[n][s][3] = a.w;
        x[n][s][4] = b.x, x[n][s][5] = b.y, x[n][s][6] = b.z, x[n][s][7] = b.w;
      }
    }
    bool far = false;
#pragma unroll
    for (uint32_t n = 0; n < NB; n++) {
      float largest = 0.f;
#pragma unroll
      for (uint32_t s = 0; s < KS; s++)
#pragma unroll
        for (int j = 0; j < 8; j++) {
          x[n][s][j] *= c2;
          largest = fmaxf(largest, fabsf(x[n][s][j]));
        }
      largest = fmaxf(largest, __shfl_xor(largest, 16, 64));
      largest = fmaxf(largest, __shfl_xor(largest, 32, 64));
      const float factor = query_factor(largest);
      far |= factor != 1.f;
      back[n] = 1.f / factor;
#pragma unroll
      for (uint32_t s = 0; s < KS; s++)
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const float v = in_f32(x[n][s][j] * factor);
          qh[n][s][j] = (_Float16)v;
          ql[n][s][j] = (_Float16)(v - (float)qh[n][s][j]);
        }
    }
    far = __builtin_amdgcn_ballot_w64(far) != 0;
    const float one = in_f32(1.f);
    af4_t o[NB][OB];
#pragma unroll
    for (uint32_t n = 0; n < NB; n++)
#pragma unroll
      for (uint32_t b = 0; b < OB; b++) o[n][b] = af4_t{0.f, 0.f, 0.f, 0.f};

    // 32 keys; `is_masked` where some row may not see them all, or has a factor.
    auto keys32 = [&](auto is_masked) __attribute__((always_inline)) {
      constexpr bool masked = decltype(is_masked)::value;
      const uint32_t next = after(step);
      const Pages coming = pages_of(after(next));
      uint32_t word[NB];  // the step's keys that a row sees
      if constexpr (masked) {
#pragma unroll
        for (uint32_t n = 0; n < NB; n++)
          word[n] = (int)(32 * step + 32) <= whole ? ~0u : tree ? trees.masks[sees_at[n] + step] : keys_to((int)(sees_at[n] - 32 * step));
      }
      // Scores of 2 x 16 keys: this lane's are 16t + 4·quad + i.
      float u[NB][2][4];
#pragma unroll
      for (int t = 0; t < 2; t++) {
        af4_t s[NB];
#pragma unroll
        for (uint32_t k = 0; k < KS; k++) {
          ah8_t a;
          if constexpr (QUANT)
            a = join(widen<FORMAT>(kr.x[t][k / 2][2 * (k % 2)]), widen<FORMAT>(kr.x[t][k / 2][2 * (k % 2) + 1]));
          else
            a = __builtin_bit_cast(ah8_t, kr.x[t][k]);
#pragma unroll
          for (uint32_t n = 0; n < NB; n++) {
            s[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qh[n][k], k ? s[n] : af4_t{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
            s[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ql[n][k], s[n], 0, 0, 0);
          }
        }
        const float ks[4] = {kr.s[t].x, kr.s[t].y, kr.s[t].z, kr.s[t].w};
#pragma unroll
        for (uint32_t n = 0; n < NB; n++) {
#pragma unroll
          for (int i = 0; i < 4; i++) {
            float x = s[n][i];
            if constexpr (masked) x *= back[n];
            u[n][t][i] = QUANT ? fmaf(x, ks[i], -m[n]) : x - m[n];
          }
        }
      }
      load(kr, pages, next, 0);
      float vs[2][4];
      float cap = 0.f;  // the largest log2 b of the lane's keys
      if constexpr (QUANT) {
#pragma unroll
        for (int t = 0; t < 2; t++) {
          vs[t][0] = vr.s[t].x, vs[t][1] = vr.s[t].y, vs[t][2] = vr.s[t].z, vs[t][3] = vr.s[t].w;
          cap = fmaxf(cap, fmaxf(fmaxf(vs[t][0], vs[t][1]), fmaxf(vs[t][2], vs[t][3])));
        }
        cap = scale_log(cap) - 127.f;
      }
      // A row's bound on u + log2 b: the largest u with the largest log2 b of the keys, which all rows see;
      // where they may not, of each key that the row sees.
      bool look = false;
      float bound[NB];
#pragma unroll
      for (uint32_t n = 0; n < NB; n++) {
        bound[n] = -INFINITY;
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            if constexpr (masked) {
              u[n][t][i] = word[n] >> (16 * t + 4 * quad + i) & 1 ? u[n][t][i] : -INFINITY;
              bound[n] = fmaxf(bound[n], QUANT ? u[n][t][i] + (scale_log(vs[t][i]) - 127.f) : u[n][t][i]);
            } else {
              bound[n] = fmaxf(bound[n], u[n][t][i]);
            }
          }
        if constexpr (!masked) bound[n] += cap;
        look |= bound[n] > lazy[n];
      }
      // Where it is past a row's limit, key by key.  That row then moves from kPeak on, so that the next
      // steps look less often.  (Other rows stay: what a row does goes by its own keys alone.)
      if (__builtin_amdgcn_ballot_w64(look)) {
#pragma unroll
        for (uint32_t n = 0; n < NB; n++) {
          auto of_row = [](float x) {
            x = fmaxf(x, __shfl_xor(x, 16, 64));
            return fmaxf(x, __shfl_xor(x, 32, 64));
          };
          auto highest = [&]() __attribute__((always_inline)) {
            float top = -INFINITY;
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
              for (int i = 0; i < 4; i++) top = fmaxf(top, QUANT ? u[n][t][i] + scale_log(vs[t][i]) : u[n][t][i]);
            return of_row(QUANT ? top - 127.f : top);
          };
          float top = highest();
          // (The same in the four lanes of a row.)
          const bool move = of_row(bound[n]) > lazy[n] && top > fminf(lazy[n], kPeak);
          const float d = move ? top - kPeak : 0.f, corr = !move || lazy[n] == kUnset ? 1.f : __builtin_amdgcn_exp2f(-d);
          m[n] += d;
          l[n] *= corr;
          lazy[n] = move ? kLazy : lazy[n];
#pragma unroll
          for (uint32_t b = 0; b < OB; b++) o[n][b] *= corr;
#pragma unroll
          for (int t = 0; t < 2; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) u[n][t][i] -= d;
          const bool coarse = fabsf(d) > kCoarse;
          if (__builtin_amdgcn_ballot_w64(coarse)) {
            top = highest();
            const float rest = coarse ? top - kPeak : 0.f;
            m[n] += rest;
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
              for (int i = 0; i < 4; i++) u[n][t][i] -= rest;
          }
        }
      }
      ah8_t ph[NB], pl[NB];
#pragma unroll
      for (uint32_t n = 0; n < NB; n++) {
        float sum = 0.f;  // of the step, so that l takes one rounding from it
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
          for (int i = 0; i < 4; i += 2) {
            const float p0 = __builtin_amdgcn_exp2f(u[n][t][i]), p1 = __builtin_amdgcn_exp2f(u[n][t][i + 1]);
            sum += p0 + p1;
            af2_t pv = {p0, p1};
            if constexpr (QUANT) {
              float b0 = vs[t][i], b1 = vs[t][i + 1];
              if constexpr (masked) {  // (a scale may be NaN, which 0 times it would be too)
                b0 = word[n] >> (16 * t + 4 * quad + i) & 1 ? b0 : 0.f;
                b1 = word[n] >> (16 * t + 4 * quad + i + 1) & 1 ? b1 : 0.f;
              }
              pv = {in_f32(p0 * b0), in_f32(p1 * b1)};
            }
            const ah2_t h = __builtin_convertvector(pv, ah2_t);
            // (One instruction each, with the f16 number as a factor, rather than its widening and a difference.)
            const af2_t rest = {fmaf(-(float)h[0], one, pv[0]), fmaf(-(float)h[1], one, pv[1])};
            const ah2_t e = __builtin_convertvector(rest, ah2_t);
            ph[n][4 * t + i] = h[0], ph[n][4 * t + i + 1] = h[1];
            pl[n][4 * t + i] = e[0], pl[n][4 * t + i + 1] = e[1];
          }
        l[n] += sum;
      }
      if constexpr (FORMAT == BCH_KV_F8) {
        // Bytes behind the last key may be NaN.  (Those of stored rows never are.)
        if (masked && 32 * step + 31 >= n_keys) {
#pragma unroll
          for (int t = 0; t < 2; t++) {
            const uint32_t keep = bytes_below((int)(n_keys - (32 * step + 16 * t + 4 * quad)));
#pragma unroll
            for (uint32_t c = 0; c < NL; c++) vr.x[t][c] &= keep;
          }
        }
      }
      // O^T += V^T·P^T: the lane's k-indices are the same 2 x 4 keys, of element 16·b + lane % 16.
#pragma unroll
      for (uint32_t b = 0; b < OB; b++) {
        const uint32_t c = b / M, x = b % M;
        ah8_t a;
        if constexpr (QUANT)
          a = join(widen<FORMAT>(vr.x[0][c][x]), widen<FORMAT>(vr.x[1][c][x]));
        else
          a = join(halves(vr.x[0][c][2 * x], vr.x[0][c][2 * x + 1]), halves(vr.x[1][c][2 * x], vr.x[1][c][2 * x + 1]));
        if constexpr (!QUANT && masked) {
          // f16 values may be infinite or NaN (k_attn_tokens): behind the last key they become 0, and rows that see
          // one get NaN from a count, with the product leaving it out.
          bool odd = false;
#pragma unroll
          for (int j = 0; j < 8; j++) {
            if (32 * step + 16 * (j / 4) + 4 * quad + j % 4 >= n_keys) a[j] = (_Float16)0.f;
            odd |= not_finite(a[j]);
          }
          if (__builtin_amdgcn_ballot_w64(odd)) {
            ah8_t bad;
#pragma unroll
            for (int j = 0; j < 8; j++) {
              bad[j] = (_Float16)(not_finite(a[j]) ? 1.f : 0.f);
              a[j] = not_finite(a[j]) ? (_Float16)0.f : a[j];
            }
#pragma unroll
            for (uint32_t n = 0; n < NB; n++) {
              ah8_t seen;
#pragma unroll
              for (int j = 0; j < 8; j++) seen[j] = (_Float16)(word[n] >> (16 * (j / 4) + 4 * quad + j % 4) & 1 ? 1.f : 0.f);
              const af4_t count = __builtin_amdgcn_mfma_f32_16x16x32_f16(bad, seen, af4_t{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
              for (int i = 0; i < 4; i++) o[n][b][i] = count[i] > 0.f ? NAN : o[n][b][i];
            }
          }
        }
#pragma unroll
        for (uint32_t n = 0; n < NB; n++) {
          o[n][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ph[n], o[n][b], 0, 0, 0);
          o[n][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, pl[n], o[n][b], 0, 0, 0);
        }
      }
      load(vr, pages, next, 1);
      pages = coming;
    };
    if (!far)
      for (; step < it.hi && (int)(32 * step + 32) <= whole; step += 4) keys32(std::false_type{});
    for (; step < it.hi; step += 4) keys32(std::true_type{});

    // Join the waves, a block of rows at a time.
#pragma unroll
    for (uint32_t n = 0; n < NB; n++) {
      l[n] += __shfl_xor(l[n], 16, 64);
      l[n] += __shfl_xor(l[n], 32, 64);
      if (quad == 0) {
        m_s[wave][col] = lazy[n] == kUnset ? -INFINITY : m[n];
        l_s[wave][col] = l[n];
      }
#pragma unroll
      for (uint32_t b = 0; b < OB; b++) *reinterpret_cast<af4_t *>(&o_s[wave][col][16 * b + 4 * quad]) = o[n][b];
      __syncthreads();
      const uint32_t rows = min(16u, it.rows - 16 * n);
      for (uint32_t i = threadIdx.x; i < rows * (HD / 4); i += 256) {
        const uint32_t row = i / (HD / 4), d = 4 * (i % (HD / 4));
        const float top = fmaxf(fmaxf(m_s[0][row], m_s[1][row]), fmaxf(m_s[2][row], m_s[3][row]));
        float4 acc = {0.f, 0.f, 0.f, 0.f};
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < 4; w++) {
          const float f = m_s[w][row] == top ? 1.f : __builtin_amdgcn_exp2f(m_s[w][row] - top);
          const float4 x = *reinterpret_cast<const float4 *>(&o_s[w][row][d]);
          acc.x = fmaf(x.x, f, acc.x), acc.y = fmaf(x.y, f, acc.y), acc.z = fmaf(x.z, f, acc.z), acc.w = fmaf(x.w, f, acc.w);
          sum = fmaf(l_s[w][row], f, sum);
        }
        const uint32_t at = it.first + 16 * n + row;
        put_row<HD>(to, it.part, kv * it.rows + 16 * n + row, it.row + at / group, kv * group + at % group, d, acc, top, sum);
      }
      __syncthreads();  // the next sums come to the same place
    }
  };
  for (uint32_t item = starts ? starts[share] : share; item < end; item++) {
    const KvAttnItem it = items[item];
    const uint32_t blocks = (it.rows + 15) / 16;
    if (MOST >= 3 && blocks == 3)
      tile(it, std::integral_constant<uint32_t, std::min(3u, MOST)>{});
    else if (MOST >= 2 && blocks == 2)
      tile(it, std::integral_constant<uint32_t, std::min(2u, MOST)>{});
    else
      tile(it, std::integral_constant<uint32_t, 1>{});
  }
}

void launch_tree_tiles(const AttnCall &a) {
  const bch_kv_plan *plan = a.plan;
  const uint32_t n_kv = plan->shape.n_kv_heads;
  const AttnTrees trees{plan->d_nodes, plan->d_masks};
  const bch_kv_plan::Work &c = plan->chunks, &t = plan->tiles16;
  kv_dispatch(plan->shape.format, plan->shape.head_dim, [&](auto format, auto hd) {
    constexpr uint32_t F = decltype(format)::value, HD = decltype(hd)::value;
    if (c.groups)
      k_attn_chunk<F, HD, true><<<c.groups * n_kv, 256, 0, a.stream>>>(a.geo, c.items, c.starts, a.q, a.q_stride, a.to,
                                                                       a.group, a.c2, trees);
    auto narrow = [&](auto most) {
      k_attn_tree<F, HD, decltype(most)::value><<<t.groups * n_kv, 256, 0, a.stream>>>(
          a.geo, t.items, t.starts, a.q, a.q_stride, a.to, a.group, a.c2, trees);
    };
    if (t.groups && plan->tree_blocks > 1)
      narrow(std::integral_constant<uint32_t, tree_most(F, HD, 2)>{});
    else if (t.groups)
      narrow(std::integral_constant<uint32_t, tree_most(F, HD, 1)>{});
  });
}

}  // namespace bch
