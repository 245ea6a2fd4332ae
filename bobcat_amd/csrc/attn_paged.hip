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
#include <algorithm>
#include <cmath>
#include <numeric>

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

// Workgroups of a CU that the registers let run at once.  (Up to 17 registers of
// the wide tiles and four of the narrow ones are spilled for it, where an item
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

template <uint32_t FORMAT, uint32_t HD>
__global__ __launch_bounds__(256, chunk_groups(FORMAT, HD)) void k_attn_chunk(
    KvGeometry g, const KvAttnItem *__restrict__ items, const uint32_t *__restrict__ starts, const float *__restrict__ q,
    uint32_t q_stride, AttnOut to, uint32_t group, float c2) {
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
    const uint32_t wg_pos0 = it.past + it.first / group;                   // the workgroup's first row's
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
      auto seen = [&](int r) __attribute__((always_inline)) { return kb + 8 * (r / 4) + 4 * half_id + r % 4 <= pos; };
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
                seen[i] = (_Float16)(kb + 16 * j + 4 * half_id + (i & 4) * 2 + (i & 3) <= pos ? 1.f : 0.f);
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
      for (; kb < hi && kb + KEYS - 1 <= wg_pos0; kb += KEYS, buf ^= 1) {
        // The other buffer was read before the last barrier.
        if (kb < last_step) {
          if (kb + 2 * KEYS - 1 <= wg_pos0)
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

KvSchedule kv_schedule(const std::vector<KvSeq> &seqs, uint32_t group, uint32_t n_kv, uint32_t format, uint32_t head_dim,
                       uint32_t n_cus, uint64_t partial_floats) {
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
  const uint32_t few_rows = wide || (large && narrow_work > kSmallBatch) ? 32 : kChunkRows;
  std::vector<Tile> narrow, tokens, chunks;
  uint32_t longest = 0;
  uint64_t narrow_steps = 0, token_steps = 0;
  for (const KvSeq &q : seqs) {
    const uint32_t rows = q.n_new * group;
    const bool few = rows <= few_rows;
    for (uint32_t first = 0; first < rows; first += few ? 16 : kChunkRows) {
      const uint32_t n = std::min(few ? 16 : kChunkRows, rows - first), keys = q.past + (first + n - 1) / group + 1;
      const Tile t{{q.table, q.past, q.row, first, n, 0, 0, ~0u}, (keys + 31) / 32};
      (!few ? chunks : n <= 8 ? narrow : tokens).push_back(t);
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
  const uint64_t few_groups = (uint64_t)n_cus * (head_dim == 256 ? 1 : token_groups(format, head_dim)) / n_kv;
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
    const KvGeometry geo = plan->geometry(cp);
    const AttnOut to{op, out_stride, ctx->attn_partials};
    const uint32_t n_kv = s.n_kv_heads, group = plan->n_heads / n_kv;
    const float c2 = (float)(1.44269504088896340736 / std::sqrt((double)s.head_dim));
    kv_dispatch(s.format, s.head_dim, [&](auto format, auto hd) {
      constexpr uint32_t F = decltype(format)::value, HD = decltype(hd)::value;
      const bch_kv_plan::Work &c = plan->chunks, &t16 = plan->tiles16, &t8 = plan->tiles8;
      if (c.groups)
        k_attn_chunk<F, HD><<<c.groups * n_kv, 256, 0, st>>>(geo, c.items, c.starts, qp, q_stride, to, group, c2);
      if (t16.groups)
        k_attn_tokens<F, HD, 16><<<t16.groups * n_kv, 256, 0, st>>>(geo, t16.items, t16.starts, qp, q_stride, to, group, c2);
      if (t8.groups)
        k_attn_tokens<F, HD, 8><<<t8.groups * n_kv, 256, 0, st>>>(geo, t8.items, t8.starts, qp, q_stride, to, group, c2);
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
