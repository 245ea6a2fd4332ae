// Attention of a batch's new tokens over the paged cache: token i of a sequence
// with `past` positions attends to positions 0 .. past + i of its pages,
// softmax(q·k/√hd)·v, with the rows that the cache holds (in the 8-bit formats
// scale·integer or scale·e4m3).
//
// The query heads of a KV head's group and a sequence's tokens are one list of
// packed rows, row = token·group + head: every row of a tile reads the same
// keys, whatever the group.  Two kernels share the mathematics:
//   k_attn_tokens: tiles of at most 16 packed rows (decoding, drafts, short
//     chunks).  A wave takes 32 keys at a time from memory straight into the
//     operands of 16x16x32 MFMAs, with no barrier in its loop; the waves of a
//     workgroup, and the pieces of a tile, have keys of their own and are joined.
//     Bound by the cache's bytes: 64 sequences of up to 16,384 int8 positions, 8
//     KV heads of 64, 99 us (5.4 TB/s; with the join 103), 16 of up to 32,768 in
//     f16 86 us; one short sequence by latency (600 positions 7.0 us).
//   k_attn_chunk: tiles of 128 packed rows, 32 a wave, that share the keys
//     through LDS.  Bound by the clock that the matrix cores' work leaves and by
//     what they wait for between the softmax's instructions: two prompts of up to
//     1,024 tokens over 16,384 int8 keys, 32 heads of 128, 780-800 us, 950-975
//     TFLOP/s (both parts counted; a large library product reaches 1,200), the
//     matrix cores busy 46% of the cycles.
// kv_schedule says which of a batch's sequences take which.
//
// Scores come as S^T = K·Q^T (keys x rows), so that a lane holds scores of one
// row, and as probabilities they are in place as an operand of O^T = V^T·P^T.
// The cache's elements are exact in f16.  Queries, taken times scale·log2 e,
// and probabilities enter as f16 high and low parts (~22 bits) and accumulate
// in f32.  With a row's key scale a and value scale b (1 in f16) and a running
// reference m,
//   u = a·s − m,  p = 2^u,  l += p,  O += (p·b)·v,
// where m follows the largest u + log2 b: p·b then stays inside f16's range,
// whatever the scales, and p needs no bound of its own (scales lie in 2^-40 ..
// 2^60).  m moves only when p·b could leave its range, so most steps rescale
// nothing.
// A plan with trees has narrow tiles of its own (attn_tree.hip) and the wide ones
// with TREE, which takes what a token sees from the plan's masks, a word for 32
// keys, in the steps with new tokens' keys; the steps of the past are the same.
#pragma once
#include <cmath>

#include "device.h"
#include "kernels.h"
#include "kv_cache.h"
#include "runtime.h"

namespace bch {

typedef _Float16 ah2_t __attribute__((ext_vector_type(2)));
typedef _Float16 ah4_t __attribute__((ext_vector_type(4)));
typedef _Float16 ah8_t __attribute__((ext_vector_type(8)));
typedef float af2_t __attribute__((ext_vector_type(2)));
typedef float af4_t __attribute__((ext_vector_type(4)));
typedef float af16_t __attribute__((ext_vector_type(16)));
typedef uint32_t au4_t __attribute__((ext_vector_type(4)));

// The reference is set so that the largest p·b is 2^kPeak, and moves when one
// passes 2^kLazy: high in f16's range, so that the low parts of much smaller
// ones are still normal numbers, with room for scale_log's error.
constexpr float kPeak = 8.f, kLazy = 14.f;
// A reference that moves further than kCoarse takes u with it only to its own last
// place, so it moves again by what is left, up or down.  (O and l are 0 then.  From
// 2^33 on the first move is the largest u itself; below, the second one's last
// place is 2^-11.)
constexpr float kCoarse = 262144.f;
constexpr float kUnset = -INFINITY;      // in its place, of a row that has seen no key yet

// Four elements of 8 bits as f16, exactly.
template <uint32_t FORMAT>
__device__ __forceinline__ ah4_t widen(uint32_t w) {
  if constexpr (FORMAT == BCH_KV_I8) {
    // Behind 0x64 the byte v + 128 is the f16 number 1024 + 128 + v.
    const uint32_t x = w ^ 0x80808080u;
    const uint32_t lo = __builtin_amdgcn_perm(0x64646464u, x, 0x04010400u);
    const uint32_t hi = __builtin_amdgcn_perm(0x64646464u, x, 0x04030402u);
    const ah2_t bias = {(_Float16)1152.f, (_Float16)1152.f};
    const ah2_t a = __builtin_bit_cast(ah2_t, lo) - bias, b = __builtin_bit_cast(ah2_t, hi) - bias;
    return {a[0], a[1], b[0], b[1]};
  } else {
    const ah2_t a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false);
    const ah2_t b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true);
    return {a[0], a[1], b[0], b[1]};
  }
}
__device__ __forceinline__ ah8_t join(ah4_t a, ah4_t b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }
__device__ __forceinline__ ah4_t halves(uint32_t a, uint32_t b) { return __builtin_bit_cast(ah4_t, ((uint64_t)b << 32) | a); }

// log2 b to within 0.09, plus 127, from a scale's bits (0 for b = 0).
__device__ __forceinline__ float scale_log(float b) { return (float)__float_as_int(b) * 0x1p-23f; }

// x as it is in f32.  A product that is then rounded to f16 may otherwise be
// rounded once, inside the multiplication, for one of its uses and twice for
// another: a high part and the low part taken from it would then not belong
// together (one element in 8,000 was off by an f16 step of its high part).
__device__ __forceinline__ float in_f32(float x) {
  asm("" : "+v"(x));
  return x;
}

__device__ __forceinline__ bool not_finite(_Float16 x) { return (__builtin_bit_cast(uint16_t, x) & 0x7c00) == 0x7c00; }

// The lowest n bytes (0 to 4, clamped).
__device__ __forceinline__ uint32_t bytes_below(int n) { return n >= 4 ? ~0u : n <= 0 ? 0u : (1u << (8 * n)) - 1; }

// A query's factor into f16's range, a power of two: 1 while its largest element
// (times scale·log2 e) lies in 2^-4 .. 2^15, where two f16 parts keep every element
// to 2^-21 of the largest (their step ends at 2^-24) at no cost; else the one that
// brings the largest to 2^14, and each score is taken back.
__device__ __forceinline__ float query_factor(float largest) {
  if ((largest >= 0.0625f && largest <= 32768.f) || largest == 0.f || !(largest <= 3.402823466e38f)) return 1.f;
  return ldexpf(1.f, min(14 - ilogbf(largest), 126));
}

// A plan's trees (kv_cache.h), of which TREE kernels take a tile's masks.
struct AttnTrees {
  const KvNode *nodes;
  const uint32_t *masks;
};
// Bits 0 .. n of 32 keys; none below 0.
__device__ __forceinline__ uint32_t keys_to(int n) { return n >= 31 ? ~0u : n < 0 ? 0u : (2u << n) - 1; }

struct AttnOut {
  float *out;       // batch rows
  uint32_t stride;
  float *partials;  // records of hd + 4 floats: O, the reference m, l
};

// One record or output quad: elements d .. d + 3 of a row with O, m and l.  An
// infinite f16 value times a probability's two parts is an infinity or, where
// the low part is 0 or of the other sign, NaN: outputs that see one are NaN
// either way.  (Nothing else makes O infinite: values are below 2^68.)
template <uint32_t HD>
__device__ __forceinline__ void put_row(const AttnOut &o, uint32_t part, uint32_t record, uint64_t row, uint32_t head, uint32_t d,
                                        float4 acc, float m, float l) {
  if (part == ~0u) {
    const float inv = 1.f / l;
    auto finite = [](float x) { return fabsf(x) <= 3.402823466e38f ? x : NAN; };
    *reinterpret_cast<float4 *>(o.out + row * o.stride + (uint64_t)head * HD + d) =
        float4{finite(acc.x * inv), finite(acc.y * inv), finite(acc.z * inv), finite(acc.w * inv)};
  } else {
    float *p = o.partials + ((uint64_t)part + record) * (HD + 4);
    *reinterpret_cast<float4 *>(p + d) = acc;
    if (d == 0) p[HD] = m, p[HD + 1] = l;
  }
}

// Workgroups of a CU that the registers let run at once.  (Up to 18 registers of
// the wide tiles, 39 with TREE, and four of the narrow ones are spilled for it, where an item
// begins and in the staging; no block with matrix instructions reloads one.)
constexpr uint32_t token_groups(uint32_t format, uint32_t hd) {
  return format == BCH_KV_F16 ? (hd == 64 ? 4 : hd == 128 ? 2 : 1) : (hd == 64 ? 4 : hd == 128 ? 3 : 2);
}
constexpr uint32_t chunk_groups(uint32_t format, uint32_t hd) {
  return hd == 64 ? (format == BCH_KV_F16 ? 2 : 3) : hd == 128 ? 2 : 1;
}

// --- tiles of at most 16 packed rows ---------------------------------------------------

// ROWS 8: the high parts of the queries and probabilities are the operands'
// columns 0..7, the low parts columns 8..15, so one MFMA does both and the
// halves of O are added once at the end.  ROWS 16: two MFMAs each.
template <uint32_t FORMAT, uint32_t HD, uint32_t ROWS>
__global__ __launch_bounds__(256, token_groups(FORMAT, HD)) void k_attn_tokens(
    KvGeometry g, const KvAttnItem *__restrict__ items, const uint32_t *__restrict__ starts, const float *__restrict__ q,
    uint32_t q_stride, AttnOut to, uint32_t group, float c2) {
  constexpr bool PACK = ROWS == 8, QUANT = FORMAT != BCH_KV_F16;
  constexpr uint32_t SIZE = kv_elem_bytes(FORMAT), BYTES = kv_block_bytes(FORMAT, HD), PART = kKvBlock * HD * SIZE;
  constexpr uint32_t NL = PART / 1024;  // KB of a block's keys, and of its values
  constexpr uint32_t KS = HD / 32, OB = HD / 16, M = 4 / SIZE;
  __shared__ __align__(16) float o_s[4][ROWS][HD];
  __shared__ float m_s[4][ROWS], l_s[4][ROWS];
  const uint32_t kv = blockIdx.x % g.n_kv, share = blockIdx.x / g.n_kv, end = starts ? starts[share + 1] : share + 1;
  for (uint32_t item = starts ? starts[share] : share; item < end; item++) {
    const KvAttnItem it = items[item];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
    const uint32_t col = lane % 16, quad = lane / 16;
    const uint32_t r = PACK ? col % 8 : col, packed = it.first + min(r, it.rows - 1);
    const uint32_t token = packed / group, head = kv * group + packed % group, pos = it.past + token;
    const uint32_t pos0 = it.past + it.first / group;                             // of the tile's first row
    const uint32_t n_keys = it.past + (it.first + it.rows - 1) / group + 1;       // of its last
    const uint32_t last = (n_keys - 1) / kKvBlock;

    struct Raw {
      au4_t x[2][NL];
      float4 s[2];
    } kr, vr;
    auto block = [&](uint32_t step, int t) {
      const uint32_t b = min(2 * step + t, last);  // (past the end: the last block, masked)
      return g.block<BYTES>(g.page(it.table, b), b, kv);
    };
    auto load = [&](Raw &raw, uint32_t step, uint32_t part) __attribute__((always_inline)) {
#pragma unroll
      for (int t = 0; t < 2; t++) {
        const uint8_t *p = block(step, t);
#pragma unroll
        for (uint32_t c = 0; c < NL; c++)
          raw.x[t][c] = *reinterpret_cast<const au4_t *>(p + part * PART + 1024 * c + 16 * lane);
        if constexpr (QUANT) raw.s[t] = *reinterpret_cast<const float4 *>(p + 2 * PART + 64 * part + 16 * quad);
      }
    };
    uint32_t step = it.lo + wave;
    const bool any = step < it.hi;
    if (any) {
      load(kr, step, 0);
      load(vr, step, 1);
    }

    // The row's elements as the keys' operand has them: k-step s of the MFMA
    // takes elements 32s + 8·quad .. + 8 (f16), or of 16-byte pieces of 8-bit
    // elements the first and then the second halves.
    ah8_t qh[KS], ql[PACK ? 1 : KS];
    float back = 1.f;
    {
      const float *qr = q + (uint64_t)(it.row + token) * q_stride + (uint64_t)head * HD;
      float x[KS][8], largest = 0.f;
#pragma unroll
      for (uint32_t s = 0; s < KS; s++) {
        const uint32_t e = QUANT ? 64 * (s / 2) + 16 * quad + 8 * (s % 2) : 32 * s + 8 * quad;
        const float4 a = *reinterpret_cast<const float4 *>(qr + e), b = *reinterpret_cast<const float4 *>(qr + e + 4);
        const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int j = 0; j < 8; j++) {
          x[s][j] = v[j] * c2;
          largest = fmaxf(largest, fabsf(x[s][j]));
        }
      }
      largest = fmaxf(largest, __shfl_xor(largest, 16, 64));
      largest = fmaxf(largest, __shfl_xor(largest, 32, 64));
      const float factor = query_factor(largest);
      back = 1.f / factor;
#pragma unroll
      for (uint32_t s = 0; s < KS; s++)
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const float v = in_f32(x[s][j] * factor);
          const _Float16 hi = (_Float16)v, lo = (_Float16)(v - (float)hi);
          if constexpr (PACK) {
            qh[s][j] = col < 8 ? hi : lo;
          } else {
            qh[s][j] = hi;
            ql[s][j] = lo;
          }
        }
    }
    const bool far = __builtin_amdgcn_ballot_w64(back != 1.f) != 0;
    const float low = col < 8 ? 0.f : 1.f;  // PACK: this lane's columns carry the low parts

    af4_t o[OB];
#pragma unroll
    for (uint32_t b = 0; b < OB; b++) o[b] = af4_t{0.f, 0.f, 0.f, 0.f};
    float m = 0.f, l = 0.f, lazy = kUnset;

    for (; step < it.hi; step += 4) {
      const uint32_t next = min(step + 4, it.hi - 1);
      // Scores of the tile's 2 x 16 keys: this lane's are 16t + 4·quad + i.
      float u[2][4];
#pragma unroll
      for (int t = 0; t < 2; t++) {
        af4_t s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (uint32_t k = 0; k < KS; k++) {
          ah8_t a;
          if constexpr (QUANT)
            a = join(widen<FORMAT>(kr.x[t][k / 2][2 * (k % 2)]), widen<FORMAT>(kr.x[t][k / 2][2 * (k % 2) + 1]));
          else
            a = __builtin_bit_cast(ah8_t, kr.x[t][k]);
          s = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qh[k], s, 0, 0, 0);
          if constexpr (!PACK) s = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ql[k], s, 0, 0, 0);
        }
        const float ks[4] = {kr.s[t].x, kr.s[t].y, kr.s[t].z, kr.s[t].w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
          float x = s[i];
          if constexpr (PACK) x += dpp<kDppRor8>(x);
          if (far) x *= back;
          u[t][i] = QUANT ? fmaf(x, ks[i], -m) : x - m;
        }
      }
      load(kr, next, 0);
      float vs[2][4];
      if constexpr (QUANT) {
#pragma unroll
        for (int t = 0; t < 2; t++) vs[t][0] = vr.s[t].x, vs[t][1] = vr.s[t].y, vs[t][2] = vr.s[t].z, vs[t][3] = vr.s[t].w;
      }
      const bool masked = 32 * step + 31 > pos0;
      if (masked) {
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const bool seen = 32 * step + 16 * t + 4 * quad + i <= pos;
            u[t][i] = seen ? u[t][i] : -INFINITY;
            if constexpr (QUANT) vs[t][i] = seen ? vs[t][i] : 0.f;
          }
      }
      auto highest = [&]() __attribute__((always_inline)) {
        float top = -INFINITY;
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
          for (int i = 0; i < 4; i++) top = fmaxf(top, QUANT ? u[t][i] + scale_log(vs[t][i]) : u[t][i]);
        return QUANT ? top - 127.f : top;
      };
      float top = highest();
      if (__builtin_amdgcn_ballot_w64(top > lazy)) {
        auto of_row = [](float x) {
          x = fmaxf(x, __shfl_xor(x, 16, 64));
          return fmaxf(x, __shfl_xor(x, 32, 64));
        };
        top = of_row(top);
        const bool move = top > lazy;  // the same in the four lanes of a row
        const float d = move ? top - kPeak : 0.f, corr = !move || lazy == kUnset ? 1.f : __builtin_amdgcn_exp2f(-d);
        m += d;
        l *= corr;
        lazy = move ? kLazy : lazy;
#pragma unroll
        for (uint32_t b = 0; b < OB; b++) o[b] *= corr;
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
          for (int i = 0; i < 4; i++) u[t][i] -= d;
        const bool coarse = fabsf(d) > kCoarse;
        if (__builtin_amdgcn_ballot_w64(coarse)) {
          top = of_row(highest());
          const float rest = coarse ? top - kPeak : 0.f;
          m += rest;
#pragma unroll
          for (int t = 0; t < 2; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) u[t][i] -= rest;
        }
      }
      ah8_t ph, pl;
      float sum = 0.f;  // of the step, so that l takes one rounding from it
#pragma unroll
      for (int t = 0; t < 2; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float p = __builtin_amdgcn_exp2f(u[t][i]);
          sum += p;
          const float pv = QUANT ? in_f32(p * vs[t][i]) : p;
          const _Float16 hi = (_Float16)pv;
          if constexpr (PACK) {
            ph[4 * t + i] = (_Float16)fmaf(-(float)hi, low, pv);
          } else {
            ph[4 * t + i] = hi;
            pl[4 * t + i] = (_Float16)(pv - (float)hi);
          }
        }
      l += sum;
      if constexpr (FORMAT == BCH_KV_F8) {
        // Bytes behind the last key may be NaN.  (Those of stored rows never are.)
        if (32 * step + 31 >= n_keys) {
#pragma unroll
          for (int t = 0; t < 2; t++) {
            const uint32_t keep = bytes_below((int)(n_keys - (32 * step + 16 * t + 4 * quad)));
#pragma unroll
            for (uint32_t c = 0; c < NL; c++) vr.x[t][c] &= keep;
          }
        }
      }
      // O^T += V^T·P^T: the lane's k-indices are the same 2 x 4 keys, of element
      // 16·b + lane % 16.
#pragma unroll
      for (uint32_t b = 0; b < OB; b++) {
        const uint32_t c = b / M, x = b % M;
        ah8_t a;
        if constexpr (QUANT)
          a = join(widen<FORMAT>(vr.x[0][c][x]), widen<FORMAT>(vr.x[1][c][x]));
        else
          a = join(halves(vr.x[0][c][2 * x], vr.x[0][c][2 * x + 1]), halves(vr.x[1][c][2 * x], vr.x[1][c][2 * x + 1]));
        if constexpr (!QUANT) {
          // f16 values may be infinite or NaN, and 0 times those is NaN: what no
          // row of the tile sees becomes 0, and what some see and others do not
          // makes NaN of the former's element below.
          if (masked) {
            bool odd = false;
#pragma unroll
            for (int j = 0; j < 8; j++) {
              if (32 * step + 16 * (j / 4) + 4 * quad + j % 4 >= n_keys) a[j] = (_Float16)0.f;
              odd |= not_finite(a[j]);
            }
            if (__builtin_amdgcn_ballot_w64(odd)) {
              ah8_t seen, bad;
#pragma unroll
              for (int j = 0; j < 8; j++) {
                seen[j] = (_Float16)(32 * step + 16 * (j / 4) + 4 * quad + j % 4 <= pos ? 1.f : 0.f);
                bad[j] = (_Float16)(not_finite(a[j]) ? 1.f : 0.f);
                a[j] = not_finite(a[j]) ? (_Float16)0.f : a[j];
              }
              const af4_t count = __builtin_amdgcn_mfma_f32_16x16x32_f16(bad, seen, af4_t{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
              for (int i = 0; i < 4; i++) o[b][i] = count[i] > 0.f ? NAN : o[b][i];
            }
          }
        }
        o[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ph, o[b], 0, 0, 0);
        if constexpr (!PACK) o[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, pl, o[b], 0, 0, 0);
      }
      load(vr, next, 1);
    }

    // Join the waves.
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if (quad == 0 && col < ROWS) {
      m_s[wave][col] = lazy == kUnset ? -INFINITY : m;
      l_s[wave][col] = l;
    }
#pragma unroll
    for (uint32_t b = 0; b < OB; b++) {
      if constexpr (PACK) {
#pragma unroll
        for (int i = 0; i < 4; i++) o[b][i] += dpp<kDppRor8>(o[b][i]);
      }
      if (col < ROWS) *reinterpret_cast<af4_t *>(&o_s[wave][col][16 * b + 4 * quad]) = o[b];
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < it.rows * (HD / 4); i += 256) {
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
      const uint32_t at = it.first + row;
      put_row<HD>(to, it.part, kv * it.rows + row, it.row + at / group, kv * group + at % group, d, acc, top, sum);
    }
    __syncthreads();  // the next item's sums come to the same place
  }
}

// --- tiles of 128 packed rows ------------------------------------------------------------------

// Keys of a step: what the registers that bring the next step's hold.
constexpr uint32_t chunk_keys(uint32_t format, uint32_t hd) { return hd == 256 || (hd == 128 && format == BCH_KV_F16) ? 32 : 64; }
constexpr uint32_t kChunkRows = 128;

template <uint32_t FORMAT, uint32_t HD, bool TREE>
__global__ __launch_bounds__(256, chunk_groups(FORMAT, HD)) void k_attn_chunk(
    KvGeometry g, const KvAttnItem *__restrict__ items, const uint32_t *__restrict__ starts, const float *__restrict__ q,
    uint32_t q_stride, AttnOut to, uint32_t group, float c2, AttnTrees trees) {
  constexpr bool QUANT = FORMAT != BCH_KV_F16;
  constexpr uint32_t SIZE = kv_elem_bytes(FORMAT), BYTES = kv_block_bytes(FORMAT, HD), PART = kKvBlock * HD * SIZE;
  constexpr uint32_t KEYS = chunk_keys(FORMAT, HD), KS = HD / 16, OB = HD / 32, M = 4 / SIZE;
  constexpr uint32_t PIECES = HD * SIZE;              // 16-byte pieces of a block's keys, and of its values
  constexpr uint32_t NP = KEYS / 16 * PIECES / 256;   // of each per thread and step
  // Keys: 8 elements of key k at slot (element / 8)·KEYS + k.  Values: the keys
  // {0..3, 8..11} + 4h of 16 keys of element d at slot (2·(key / 16) + h)·HD + d.
  __shared__ __align__(16) _Float16 k_s[2][KEYS * HD], v_s[2][KEYS * HD];
  __shared__ __align__(16) float s_s[2][2][KEYS];         // the keys' and the values' scales
  __shared__ float top_s[2][KEYS / kKvBlock];             // the largest scale_log of each block's values
  __shared__ uint32_t odd_s[2];
  const uint32_t kv = blockIdx.x % g.n_kv, share = blockIdx.x / g.n_kv, end = starts ? starts[share + 1] : share + 1;
  for (uint32_t item = starts ? starts[share] : share; item < end; item++) {
    const KvAttnItem it = items[item];
    const uint32_t tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64) & 3, lane = tid % 64;
    const uint32_t col = lane % 32, half_id = lane / 32;
    const bool active = 32 * wave < it.rows;
    const uint32_t row0 = it.first + (active ? 32 * wave : 0);
    const uint32_t rows = active ? min(32u, it.rows - 32 * wave) : 1;
    const uint32_t packed = row0 + min(col, rows - 1);
    const uint32_t token = packed / group, head = kv * group + packed % group, pos = it.past + token;
    const uint32_t kend = it.past + (row0 + rows - 1) / group + 1;         // keys of the wave's last row
    // Keys that every row of the workgroup sees, and where the row's mask has key 0.
    int whole = it.past + it.first / group + 1;
    bool tree = false;
    const uint32_t *mask = nullptr;
    if constexpr (TREE) {
      tree = trees.nodes[it.row].mask != kKvNone;
      whole = tree ? it.past : whole;
      mask = trees.masks + (tree ? (int64_t)trees.nodes[it.row + token].mask - it.past / 32 : 0);
    }
    const uint32_t wg_kend = it.past + (it.first + it.rows - 1) / group + 1;
    const uint32_t last = (wg_kend - 1) / kKvBlock;
    const uint32_t lo = it.lo * 32, hi = min(it.hi * 32, wg_kend);         // keys of this split

    au4_t kr[NP], vr[NP];
    float scale = 0.f;  // of wave w: lanes 0..15 the key scales of block w of the step, 16..31 the value scales
    // Lanes of a value piece: quads of keys in the order 0, 2, 1, 3, so that the
    // two quads whose halves of a slot interleave are written together.
    const uint32_t swapped = (lane & 15) | (lane & 16) << 1 | (lane & 32) >> 1;
    auto block_at = [&](uint32_t b) { return g.block<BYTES>(g.page(it.table, min(b, last)), min(b, last), kv); };
    // This wave's pieces of part p are within .. + 64 of block j of the step.
    auto part_block = [&](uint32_t p) { return 64 * wave / PIECES + 256 * p / PIECES; };
    auto part_within = [&](uint32_t p) { return 64 * wave % PIECES + 256 * p % PIECES; };
    auto load = [&](uint32_t kb) __attribute__((always_inline)) {
#pragma unroll
      for (uint32_t p = 0; p < NP; p++) {
        const uint32_t j = part_block(p), within = part_within(p);
        const uint8_t *b = block_at(kb / kKvBlock + j);
        kr[p] = *reinterpret_cast<const au4_t *>(b + 16 * (within + lane));
        vr[p] = *reinterpret_cast<const au4_t *>(b + PART + 16 * (within + swapped));
      }
      if constexpr (QUANT) {
        if (wave < KEYS / kKvBlock && lane < 32)
          scale = reinterpret_cast<const float *>(block_at(kb / kKvBlock + wave) + 2 * PART)[lane];
      }
    };
    // With `ends`, keys behind the last are cleared where they could be NaN, and
    // f16 values that are not finite noted.
    auto stage = [&](int buf, uint32_t kb, auto at_end) __attribute__((always_inline)) {
      constexpr bool ends = decltype(at_end)::value;
      bool odd = false;
#pragma unroll
      for (uint32_t p = 0; p < NP; p++) {
        const uint32_t j = part_block(p), within = part_within(p);
        const uint32_t piece = within / 16 + lane / 16, key = 16 * j + lane % 16;
        if constexpr (QUANT) {
          *reinterpret_cast<ah8_t *>(&k_s[buf][(2 * piece * KEYS + key) * 8]) = join(widen<FORMAT>(kr[p][0]), widen<FORMAT>(kr[p][1]));
          *reinterpret_cast<ah8_t *>(&k_s[buf][((2 * piece + 1) * KEYS + key) * 8]) = join(widen<FORMAT>(kr[p][2]), widen<FORMAT>(kr[p][3]));
        } else {
          *reinterpret_cast<au4_t *>(&k_s[buf][(piece * KEYS + key) * 8]) = kr[p];
        }
        const uint32_t quad = swapped / 16;
        // Bytes behind the last key may be NaN.  (Those of stored rows never are.)
        if constexpr (FORMAT == BCH_KV_F8 && ends) {
          if (kb + KEYS > wg_kend) vr[p] &= bytes_below((int)(wg_kend - (kb + 16 * j + 4 * quad)));
        }
#pragma unroll
        for (uint32_t x = 0; x < M; x++) {
          const uint32_t d = within / 4 * M + 16 * x + lane % 16;
          ah4_t a;
          if constexpr (QUANT)
            a = widen<FORMAT>(vr[p][x]);
          else
            a = halves(vr[p][2 * x], vr[p][2 * x + 1]);
          if constexpr (!QUANT && ends) {
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) {
              if (kb + 16 * j + 4 * quad + i >= wg_kend) a[i] = (_Float16)0.f;
              odd |= not_finite(a[i]);
            }
          }
          *reinterpret_cast<ah4_t *>(&v_s[buf][((2 * j + quad % 2) * HD + d) * 8 + quad / 2 * 4]) = a;
        }
      }
      if constexpr (QUANT) {
        if (wave < KEYS / kKvBlock && lane < 32) {
          const float x = ends && lane >= 16 && kb + 16 * wave + lane % 16 >= wg_kend ? 0.f : scale;
          s_s[buf][lane / 16][16 * wave + lane % 16] = x;
          float top = x == x ? scale_log(x) : 0.f;
          top = fmaxf(top, dpp<kDppXor1>(top));
          top = fmaxf(top, dpp<kDppXor2>(top));
          top = fmaxf(top, dpp<kDppHalfMirror>(top));
          top = fmaxf(top, dpp<kDppMirror>(top));
          if (lane == 16) top_s[buf][wave] = top - 127.f;
        }
      } else if constexpr (ends) {
        if (__builtin_amdgcn_ballot_w64(odd) && lane == 0) odd_s[buf] = 1;  // (cleared after the step)
      }
    };
    if (tid < 2) odd_s[tid] = 0;
    if (lo < hi) load(lo);

    ah8_t qh[KS], ql[KS];
    float back = 1.f;
    {
      const float *qr = q + (uint64_t)(it.row + token) * q_stride + (uint64_t)head * HD + 8 * half_id;
      auto take = [&](float factor) __attribute__((always_inline)) {
        float largest = 0.f;
#pragma unroll
        for (uint32_t s = 0; s < KS; s++) {
          const float4 a = *reinterpret_cast<const float4 *>(qr + 16 * s), b = *reinterpret_cast<const float4 *>(qr + 16 * s + 4);
          const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
          for (int j = 0; j < 8; j++) {
            const float x = in_f32(v[j] * c2 * factor);
            largest = fmaxf(largest, fabsf(x));
            qh[s][j] = (_Float16)x;
            ql[s][j] = (_Float16)(x - (float)qh[s][j]);
          }
        }
        return fmaxf(largest, __shfl_xor(largest, 32, 64));
      };
      const float factor = query_factor(take(1.f));
      if (__builtin_amdgcn_ballot_w64(factor != 1.f)) {
        take(factor);
        back = 1.f / factor;
      }
    }
    const bool far = __builtin_amdgcn_ballot_w64(back != 1.f) != 0;
    af16_t o[OB];
#pragma unroll
    for (uint32_t b = 0; b < OB; b++)
#pragma unroll
      for (int i = 0; i < 16; i++) o[b][i] = 0.f;
    float m = 0.f, l = 0.f, lazy = kUnset;

    // 32 keys of a step from key kb on, in LDS from key k0 on; score r is of key
    // kb + 8·(r / 4) + 4·half + r % 4.
    auto tile = [&](uint32_t kb, uint32_t k0, int buf, auto is_masked) __attribute__((always_inline)) {
      constexpr bool masked = decltype(is_masked)::value;
      uint32_t word = 0;  // the 32 keys that the row sees
      if constexpr (TREE && masked)
        word = !tree ? keys_to((int)(pos - kb)) : kb + 31 < it.past ? ~0u : mask[kb / 32];
      af16_t u;
#pragma unroll
      for (int i = 0; i < 16; i++) u[i] = 0.f;
#pragma unroll
      for (uint32_t s = 0; s < KS; s++) {
        const ah8_t a = *reinterpret_cast<const ah8_t *>(&k_s[buf][((2 * s + half_id) * KEYS + k0 + col) * 8]);
        u = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qh[s], u, 0, 0, 0);
        u = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, ql[s], u, 0, 0, 0);
      }
      // The values' operands come while the softmax is computed (heads of 256
      // have no registers for them).
      auto value = [&](int j, uint32_t b) __attribute__((always_inline)) {
        return *reinterpret_cast<const ah8_t *>(&v_s[buf][((k0 / 8 + 2 * j + half_id) * HD + 32 * b + col) * 8]);
      };
      ah8_t v[2][HD == 256 ? 1 : OB];
      if constexpr (HD != 256) {
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
          for (uint32_t b = 0; b < OB; b++) v[j][b] = value(j, b);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (far) {
#pragma unroll
        for (int r = 0; r < 16; r++) u[r] *= back;
      }
      auto scales = [&](const float *from, int q4) __attribute__((always_inline)) {
        const float4 a = *reinterpret_cast<const float4 *>(from + k0 + 8 * q4 + 4 * half_id);
        return af4_t{a.x, a.y, a.z, a.w};
      };
      auto sees = [&](uint32_t key) __attribute__((always_inline)) {  // of the 32
        if constexpr (TREE) return (word >> key & 1) != 0;
        return kb + key <= pos;
      };
      auto seen = [&](int r) __attribute__((always_inline)) { return sees(8 * (r / 4) + 4 * half_id + r % 4); };
#pragma unroll
      for (int q4 = 0; q4 < 4; q4++) {
        af4_t a;
        if constexpr (QUANT) a = scales(s_s[buf][0], q4);
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int r = 4 * q4 + i;
          u[r] = QUANT ? fmaf(u[r], a[i], -m) : u[r] - m;
          if constexpr (masked) u[r] = seen(r) ? u[r] : -INFINITY;
        }
      }
      // The largest u + log2 b of this lane's keys.
      auto highest = [&]() __attribute__((always_inline)) {
        float top = -INFINITY;
#pragma unroll
        for (int q4 = 0; q4 < 4; q4++) {
          af4_t b;
          if constexpr (QUANT) b = scales(s_s[buf][1], q4);
#pragma unroll
          for (int i = 0; i < 4; i++) top = fmaxf(top, QUANT ? u[4 * q4 + i] + scale_log(b[i]) : u[4 * q4 + i]);
        }
        return QUANT ? top - 127.f : top;
      };
      // Where all keys are seen, the largest u and the largest log2 b of the tile
      // bound it and save the keys' own scales.  The bound only says where to
      // look: a reference that followed it would rise with the scale of a row that
      // no query sees much of, for good, and the others' p·b would fall out of
      // f16's range.  Every row that is past kPeak then moves, so that the next
      // steps look less often (1,024 tokens of two prompts over 4,000 keys, int8,
      // heads of 256: 173 us, 182 where only rows past kLazy move; a reference
      // that follows the bound 175).
      constexpr bool bounded = QUANT && !masked;
      auto of_row = [](float x) { return fmaxf(x, __shfl_xor(x, 32, 64)); };
      float top = -INFINITY;
      if constexpr (bounded) {
#pragma unroll
        for (int r = 0; r < 16; r++) top = fmaxf(top, u[r]);
        top += fmaxf(top_s[buf][k0 / 16], top_s[buf][k0 / 16 + 1]);
      } else {
        top = highest();
      }
      if (__builtin_amdgcn_ballot_w64(top > lazy)) {
        top = of_row(bounded ? highest() : top);
        const bool move = top > (bounded ? fminf(lazy, kPeak) : lazy);  // the same in both lanes of a row
        const float d = move ? top - kPeak : 0.f, corr = !move || lazy == kUnset ? 1.f : __builtin_amdgcn_exp2f(-d);
        m += d;
        l *= corr;
        lazy = move ? kLazy : lazy;
#pragma unroll
        for (uint32_t b = 0; b < OB; b++)
#pragma unroll
          for (int i = 0; i < 16; i++) o[b][i] *= corr;
#pragma unroll
        for (int r = 0; r < 16; r++) u[r] -= d;
        const bool coarse = fabsf(d) > kCoarse;
        if (__builtin_amdgcn_ballot_w64(coarse)) {
          top = of_row(highest());
          const float rest = coarse ? top - kPeak : 0.f;
          m += rest;
#pragma unroll
          for (int r = 0; r < 16; r++) u[r] -= rest;
        }
      }
      ah8_t ph[2], pl[2];
      float sum = 0.f;  // of the tile, so that l takes one rounding from it
#pragma unroll
      for (int q4 = 0; q4 < 4; q4++) {
        af4_t b;
        if constexpr (QUANT) b = scales(s_s[buf][1], q4);
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          const int r = 4 * q4 + i;
          const float p0 = __builtin_amdgcn_exp2f(u[r]), p1 = __builtin_amdgcn_exp2f(u[r + 1]);
          sum += p0 + p1;
          af2_t pv = {p0, p1};
          if constexpr (QUANT) {
            // (A scale may be NaN, which 0 times it would be too.)
            if constexpr (masked) b[i] = seen(r) ? b[i] : 0.f, b[i + 1] = seen(r + 1) ? b[i + 1] : 0.f;
            pv = {in_f32(p0 * b[i]), in_f32(p1 * b[i + 1])};
          }
          const ah2_t h = __builtin_convertvector(pv, ah2_t);
          const af2_t rest = {pv[0] - (float)h[0], pv[1] - (float)h[1]};
          const ah2_t e = __builtin_convertvector(rest, ah2_t);
          ph[r / 8][r % 8] = h[0], ph[r / 8][r % 8 + 1] = h[1];
          pl[r / 8][r % 8] = e[0], pl[r / 8][r % 8 + 1] = e[1];
        }
      }
      l += sum;
#pragma unroll
      for (int j = 0; j < 2; j++)
#pragma unroll
        for (uint32_t b = 0; b < OB; b++) {
          ah8_t a = HD == 256 ? value(j, b) : v[j][HD == 256 ? 0 : b];
          if constexpr (masked && !QUANT) {
            // 0 times a value that is not finite is NaN: rows that see such a
            // value get it from a count, and the product leaves it out.
            if (odd_s[buf]) {
              ah8_t seen, bad;
              af16_t count;
#pragma unroll
              for (int i = 0; i < 16; i++) count[i] = 0.f;
#pragma unroll
              for (int i = 0; i < 8; i++) {
                seen[i] = (_Float16)(sees(16 * j + 4 * half_id + (i & 4) * 2 + (i & 3)) ? 1.f : 0.f);
                bad[i] = (_Float16)(not_finite(a[i]) ? 1.f : 0.f);
                a[i] = not_finite(a[i]) ? (_Float16)0.f : a[i];
              }
              count = __builtin_amdgcn_mfma_f32_32x32x16_f16(bad, seen, count, 0, 0, 0);
#pragma unroll
              for (int i = 0; i < 16; i++) o[b][i] = count[i] > 0.f ? NAN : o[b][i];
            }
          }
          o[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, ph[j], o[b], 0, 0, 0);
          o[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, pl[j], o[b], 0, 0, 0);
        }
    };
    if (lo < hi) {
      const uint32_t last_step = (hi - 1) / KEYS * KEYS;
      __syncthreads();  // odd_s is clear
      stage(0, lo, std::true_type{});
      load(min(lo + KEYS, last_step));
      lds_barrier();
      uint32_t kb = lo;
      int buf = 0;
      // Steps that every row sees whole.
      for (; kb < hi && (int)(kb + KEYS) <= whole; kb += KEYS, buf ^= 1) {
        // The other buffer was read before the last barrier.
        if (kb < last_step) {
          if ((int)(kb + 2 * KEYS) <= whole)
            stage(buf ^ 1, kb + KEYS, std::false_type{});
          else
            stage(buf ^ 1, kb + KEYS, std::true_type{});
          load(min(kb + 2 * KEYS, last_step));
        }
        if (active) {
#pragma unroll 1
          for (uint32_t k0 = 0; k0 < KEYS; k0 += 32) tile(kb + k0, k0, buf, std::false_type{});
        }
        lds_barrier();
      }
      // The others.
      for (; kb < hi; kb += KEYS, buf ^= 1) {
        if (kb < last_step) {
          stage(buf ^ 1, kb + KEYS, std::true_type{});
          load(min(kb + 2 * KEYS, last_step));
        }
        if (active) {
#pragma unroll 1
          for (uint32_t k0 = 0; k0 < KEYS && kb + k0 < kend; k0 += 32) tile(kb + k0, k0, buf, std::true_type{});
        }
        lds_barrier();
        if constexpr (!QUANT) {
          if (tid == 0) odd_s[buf] = 0;
          lds_barrier();
        }
      }
    }
    // (Every wave has passed the last step's barrier: the next item may write to
    // the stages.)
    l += __shfl_xor(l, 32, 64);
    if (active && col < rows) {
      const float ref = lazy == kUnset ? -INFINITY : m;
#pragma unroll
      for (uint32_t b = 0; b < OB; b++)
#pragma unroll
        for (int q4 = 0; q4 < 4; q4++)
          put_row<HD>(to, it.part, kv * it.rows + (packed - it.first), it.row + token, head, 32 * b + 8 * q4 + 4 * half_id,
                      float4{o[b][4 * q4], o[b][4 * q4 + 1], o[b][4 * q4 + 2], o[b][4 * q4 + 3]}, ref, l);
    }
  }
}

// An attention call's operands, and attn_tree.hip's launches for a plan with trees
// (all but the join): its tiles16 are tiles of up to tree_tile_rows rows.
struct AttnCall {
  hipStream_t stream;
  const bch_kv_plan *plan;
  KvGeometry geo;
  const float *q;
  uint32_t q_stride, group;
  AttnOut to;
  float c2;
};
void launch_tree_tiles(const AttnCall &a);
uint32_t tree_tile_rows(uint32_t format, uint32_t hd);
uint32_t tree_tile_groups(uint32_t format, uint32_t hd, uint32_t blocks);  // workgroups of a CU

}  // namespace bch
