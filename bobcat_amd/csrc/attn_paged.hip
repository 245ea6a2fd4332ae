// Attention of a batch's new tokens over the paged cache: token i of a sequence
// with `past` positions attends to positions 0 .. past + i of its pages,
// softmax(q·k/√hd)·v, with the rows that the cache holds (in the 8-bit formats
// scale·integer or scale·e4m3).
//
// The query heads of a KV head's group and a sequence's tokens are one list of
// packed rows, row = token·group + head: every row of a tile reads the same
// keys, whatever the group.  Two kernels share the mathematics:
//   k_attn_tokens: sequences of at most 16 packed rows (decoding, drafts).  A
//     wave takes 32 keys at a time from memory straight into the operands of
//     16x16x32 MFMAs; the waves of a workgroup, and the splits of a sequence,
//     have keys of their own and are joined.  Bound by the cache's bytes.
//   k_attn_chunk: tiles of 128 packed rows, 32 a wave, that share the keys
//     through LDS.  Bound by the matrix cores and the softmax's instructions.
// (The rule: with 16 rows or fewer the narrow tile wastes no matrix work and
// needs no barrier; above, the wide one reads the cache once for 128 rows.)
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
// 2^60).  m moves only when p·b would leave its range, so most steps rescale
// nothing.
#include <algorithm>
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

__device__ __forceinline__ bool not_finite(_Float16 x) { return (__builtin_bit_cast(uint16_t, x) & 0x7c00) == 0x7c00; }

// The lowest n bytes (0 to 4, clamped).
__device__ __forceinline__ uint32_t bytes_below(int n) { return n >= 4 ? ~0u : n <= 0 ? 0u : (1u << (8 * n)) - 1; }

// A query's factor to and from f16's range: 1 unless its largest element
// (times scale·log2 e) passes 2^15.
__device__ __forceinline__ float query_down(float largest) {
  if (!(largest > 32768.f) || !(largest <= 3.402823466e38f)) return 1.f;
  return __int_as_float((127 + 14 - ((__float_as_int(largest) >> 23) - 127)) << 23);
}

struct AttnOut {
  float *out;       // batch rows
  uint32_t stride;
  float *partials;  // records of hd + 4 floats: O, the reference m, l
};

// One record or output quad: elements d .. d + 3 of a row with O, m and l.
template <uint32_t HD>
__device__ __forceinline__ void put_row(const AttnOut &o, uint32_t part, uint32_t record, uint64_t row, uint32_t head, uint32_t d,
                                        float4 acc, float m, float l) {
  if (part == ~0u) {
    const float inv = 1.f / l;
    *reinterpret_cast<float4 *>(o.out + row * o.stride + (uint64_t)head * HD + d) =
        float4{acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
  } else {
    float *p = o.partials + ((uint64_t)part + record) * (HD + 4);
    *reinterpret_cast<float4 *>(p + d) = acc;
    if (d == 0) p[HD] = m, p[HD + 1] = l;
  }
}

// Workgroups of a CU that the registers let run at once.
constexpr uint32_t token_groups(uint32_t format, uint32_t hd) {
  return format == BCH_KV_F16 ? (hd == 64 ? 4 : hd == 128 ? 2 : 1) : (hd == 64 ? 4 : hd == 128 ? 3 : 2);
}
constexpr uint32_t chunk_groups(uint32_t hd) { return hd == 64 ? 3 : hd == 128 ? 2 : 1; }

// --- at most 16 packed rows ---------------------------------------------------

// ROWS 8: the high parts of the queries and probabilities are the operands'
// columns 0..7, the low parts columns 8..15, so one MFMA does both and the
// halves of O are added once at the end.  ROWS 16: two MFMAs each.
template <uint32_t FORMAT, uint32_t HD, uint32_t ROWS>
__global__ __launch_bounds__(256, token_groups(FORMAT, HD)) void k_attn_tokens(
    KvGeometry g, const KvAttnItem *__restrict__ items,
                                                                       const uint32_t *__restrict__ starts,
                                                                       const float *__restrict__ q, uint32_t q_stride,
                                                                       AttnOut to, uint32_t group, float c2) {
  constexpr bool PACK = ROWS == 8, QUANT = FORMAT != BCH_KV_F16;
  constexpr uint32_t SIZE = kv_elem_bytes(FORMAT), BYTES = kv_block_bytes(FORMAT, HD), PART = kKvBlock * HD * SIZE;
  constexpr uint32_t NL = PART / 1024;  // KB of a block's keys, and of its values
  constexpr uint32_t KS = HD / 32, OB = HD / 16, M = 4 / SIZE;
  __shared__ __align__(16) float o_s[4][ROWS][HD];
  __shared__ float m_s[4][ROWS], l_s[4][ROWS];
  const uint32_t kv = blockIdx.x % g.n_kv, end = starts[blockIdx.x / g.n_kv + 1];
  for (uint32_t item = starts[blockIdx.x / g.n_kv]; item < end; item++) {
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
  // (Past the end: the last block, masked.)  The pages are looked up a step
  // before their blocks are loaded.
  auto number = [&](uint32_t step, int t) { return min(2 * step + t, last); };
  uint32_t page[2];
  auto look_up = [&](uint32_t step) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < 2; t++) page[t] = g.page(it.table, number(step, t));
  };
  auto load = [&](Raw &raw, uint32_t step, uint32_t part) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < 2; t++) {
      const uint8_t *p = g.block<BYTES>(page[t], number(step, t), kv);
#pragma unroll
      for (uint32_t c = 0; c < NL; c++)
        raw.x[t][c] = *reinterpret_cast<const au4_t *>(p + part * PART + 1024 * c + 16 * lane);
      if constexpr (QUANT) raw.s[t] = *reinterpret_cast<const float4 *>(p + 2 * PART + 64 * part + 16 * quad);
    }
  };
  uint32_t step = it.lo + wave;
  auto after = [&](uint32_t step) { return min(step + 4, it.hi - 1); };
  if (step < it.hi) {
    look_up(step);
    load(kr, step, 0);
    load(vr, step, 1);
    look_up(after(step));
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
    const float down = query_down(largest);
    back = 1.f / down;
#pragma unroll
    for (uint32_t s = 0; s < KS; s++)
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const float v = x[s][j] * down;
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
    const uint32_t next = after(step);
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
    float top = -INFINITY;
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int i = 0; i < 4; i++) top = fmaxf(top, QUANT ? u[t][i] + scale_log(vs[t][i]) : u[t][i]);
    if constexpr (QUANT) top -= 127.f;
    if (__builtin_amdgcn_ballot_w64(top > lazy)) {
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
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
    }
    ah8_t ph, pl;
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float p = __builtin_amdgcn_exp2f(u[t][i]);
        l += p;
        const float pv = QUANT ? p * vs[t][i] : p;
        const _Float16 hi = (_Float16)pv;
        if constexpr (PACK) {
          ph[4 * t + i] = (_Float16)fmaf(-(float)hi, low, pv);
        } else {
          ph[4 * t + i] = hi;
          pl[4 * t + i] = (_Float16)(pv - (float)hi);
        }
      }
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
    look_up(after(next));
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

// --- more rows ------------------------------------------------------------------

constexpr uint32_t kChunkRows = 128;

// Steps of 32 keys, one behind the other: while a wave turns the scores of step
// t into probabilities, the matrix cores compute those of step t + 1, and while
// they multiply step t's values, it stages later keys and values in LDS.  (A
// 32x32x16 MFMA takes 32 cycles of the matrix core and leaves the wave free for
// about six other instructions; one wave's MFMAs and another's vector
// instructions hardly overlap by themselves.  With both in one stream ... us,
// apart ... for attend_mixed's chunks.)
template <uint32_t FORMAT, uint32_t HD>
__global__ __launch_bounds__(256, chunk_groups(HD)) void k_attn_chunk(
    KvGeometry g, const KvAttnItem *__restrict__ items, const uint32_t *__restrict__ starts, const float *__restrict__ q,
    uint32_t q_stride, AttnOut to, uint32_t group, float c2) {
  constexpr bool QUANT = FORMAT != BCH_KV_F16;
  constexpr uint32_t SIZE = kv_elem_bytes(FORMAT), BYTES = kv_block_bytes(FORMAT, HD), PART = kKvBlock * HD * SIZE;
  constexpr uint32_t KS = HD / 16, OB = HD / 32, M = 4 / SIZE;
  constexpr uint32_t PIECES = HD * SIZE;        // 16-byte pieces of a block's keys, and of its values
  constexpr bool SHARED = 2 * PIECES < 256;     // a step's keys are half the waves' pieces, its values the others'
  constexpr uint32_t NP = SHARED ? 1 : 2 * PIECES / 256;  // of each per thread and step
  // Keys: 8 elements of key k at slot (element / 8)·32 + k.  Values: the keys
  // {0..3, 8..11} + 4h of 16 keys of element d at slot (2·(key / 16) + h)·HD + d.
  // Those of step t lie in buffer t % 2.
  __shared__ __align__(16) _Float16 k_s[2][32 * HD], v_s[2][32 * HD];
  __shared__ __align__(16) float s_s[2][2][32];           // the keys' and the values' scales
  __shared__ float top_s[2][2];                           // the largest scale_log of each block's values
  __shared__ uint32_t odd_s[2][4];                        // of each wave: its f16 values were not all finite
  const uint32_t kv = blockIdx.x % g.n_kv, end = starts[blockIdx.x / g.n_kv + 1];
  for (uint32_t item = starts[blockIdx.x / g.n_kv]; item < end; item++) {
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
  const uint32_t last = (wg_kend - 1) / kKvBlock, last_step = it.hi - 1;

  au4_t kr[NP], vr[SHARED ? 1 : NP];
  float scale = 0.f;  // of wave w < 2: lanes 0..15 the key scales of block w of the step, 16..31 the value scales
  // Lanes of a value piece: quads of keys in the order 0, 2, 1, 3, so that the
  // two quads whose halves of a slot interleave are written together.
  const uint32_t swapped = (lane & 15) | (lane & 16) << 1 | (lane & 32) >> 1;
  // This wave's pieces of part p are within .. + 64 of block j of the step.
  const uint32_t wave_of = SHARED ? wave & 1 : wave;
  const bool keys_here = !SHARED || wave < 2, values_here = !SHARED || wave >= 2;
  auto part_block = [&](uint32_t p) { return 64 * wave_of / PIECES + 256 * p / PIECES; };
  auto part_within = [&](uint32_t p) { return 64 * wave_of % PIECES + 256 * p % PIECES; };
  // (Past the end: the last step and block again.)  The pages of the keys of
  // step n are looked up before those are loaded, and kept for its values.
  auto clamp = [&](uint32_t step) { return min(step, last_step); };
  auto number = [&](uint32_t step, uint32_t j) { return min(2 * clamp(step) + j, last); };
  uint32_t page[NP], page_before[NP], scale_page = 0;
  auto look_up = [&](uint32_t step) __attribute__((always_inline)) {
#pragma unroll
    for (uint32_t p = 0; p < NP; p++) {
      page_before[p] = page[p];
      page[p] = g.page(it.table, number(step, part_block(p)));
    }
    if constexpr (QUANT) scale_page = g.page(it.table, number(step - 1, wave & 1));
  };
  // The keys of step n and the values of step n - 1.
  auto load_keys = [&](uint32_t step) __attribute__((always_inline)) {
    if (!keys_here) return;
#pragma unroll
    for (uint32_t p = 0; p < NP; p++)
      kr[p] = *reinterpret_cast<const au4_t *>(g.block<BYTES>(page[p], number(step, part_block(p)), kv) +
                                               16 * (part_within(p) + lane));
  };
  auto load_values = [&](uint32_t step) __attribute__((always_inline)) {
    if (values_here) {
#pragma unroll
      for (uint32_t p = 0; p < NP; p++)
        (SHARED ? kr : vr)[p] = *reinterpret_cast<const au4_t *>(g.block<BYTES>(page_before[p], number(step, part_block(p)), kv) +
                                                                 PART + 16 * (part_within(p) + swapped));
    }
    if constexpr (QUANT) {
      if (wave < 2 && lane < 32)
        scale = reinterpret_cast<const float *>(g.block<BYTES>(scale_page, number(step, wave), kv) + 2 * PART)[lane];
    }
  };
  auto stage_keys = [&](uint32_t buf) __attribute__((always_inline)) {
    if (!keys_here) return;
#pragma unroll
    for (uint32_t p = 0; p < NP; p++) {
      const uint32_t piece = part_within(p) / 16 + lane / 16, key = 16 * part_block(p) + lane % 16;
      if constexpr (QUANT) {
        *reinterpret_cast<ah8_t *>(&k_s[buf][(2 * piece * 32 + key) * 8]) = join(widen<FORMAT>(kr[p][0]), widen<FORMAT>(kr[p][1]));
        *reinterpret_cast<ah8_t *>(&k_s[buf][((2 * piece + 1) * 32 + key) * 8]) = join(widen<FORMAT>(kr[p][2]), widen<FORMAT>(kr[p][3]));
      } else {
        *reinterpret_cast<au4_t *>(&k_s[buf][(piece * 32 + key) * 8]) = kr[p];
      }
    }
  };
  // With `ends`, values behind the last key are cleared where they could be NaN,
  // and f16 values that are not finite noted.
  auto stage_values = [&](uint32_t buf, uint32_t kb, auto at_end) __attribute__((always_inline)) {
    constexpr bool ends = decltype(at_end)::value;
    bool odd = false;
    if (values_here) {
#pragma unroll
      for (uint32_t p = 0; p < NP; p++) {
        const uint32_t j = part_block(p), quad = swapped / 16;
        au4_t x = (SHARED ? kr : vr)[p];
        // Bytes behind the last key may be NaN.  (Those of stored rows never are.)
        if constexpr (FORMAT == BCH_KV_F8 && ends) x &= bytes_below((int)(wg_kend - (kb + 16 * j + 4 * quad)));
#pragma unroll
        for (uint32_t e = 0; e < M; e++) {
          const uint32_t d = part_within(p) / 4 * M + 16 * e + lane % 16;
          ah4_t a;
          if constexpr (QUANT)
            a = widen<FORMAT>(x[e]);
          else
            a = halves(x[2 * e], x[2 * e + 1]);
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
    }
    if constexpr (QUANT) {
      if (wave < 2 && lane < 32) {
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
      const bool any = __builtin_amdgcn_ballot_w64(odd) != 0;
      if (lane == 0) odd_s[buf][wave] = any;
    }
  };
#pragma unroll
  for (uint32_t p = 0; p < NP; p++) page[p] = 0;
  look_up(it.lo);
  load_keys(it.lo);

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
          const float x = v[j] * c2 * factor;
          largest = fmaxf(largest, fabsf(x));
          qh[s][j] = (_Float16)x;
          ql[s][j] = (_Float16)(x - (float)qh[s][j]);
        }
      }
      return fmaxf(largest, __shfl_xor(largest, 32, 64));
    };
    const float down = query_down(take(1.f));
    if (__builtin_amdgcn_ballot_w64(down != 1.f)) {
      take(down);
      back = 1.f / down;
    }
  }
  const bool far = __builtin_amdgcn_ballot_w64(back != 1.f) != 0;
  af16_t o[OB], u;
#pragma unroll
  for (uint32_t b = 0; b < OB; b++)
#pragma unroll
    for (int i = 0; i < 16; i++) o[b][i] = 0.f;
  float m = 0.f, l = 0.f, lazy = kUnset;

  // S^T = K·Q^T of the keys in buffer `buf`: element r is the score of key 8·(r / 4)
  // + 4·half + r % 4 of the step.
  auto scores = [&](uint32_t buf) __attribute__((always_inline)) {
    af16_t x;
#pragma unroll
    for (int i = 0; i < 16; i++) x[i] = 0.f;
#pragma unroll
    for (uint32_t s = 0; s < KS; s++) {
      const ah8_t a = *reinterpret_cast<const ah8_t *>(&k_s[buf][((2 * s + half_id) * 32 + col) * 8]);
      x = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qh[s], x, 0, 0, 0);
      x = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, ql[s], x, 0, 0, 0);
    }
    return x;
  };
  auto scales = [&](uint32_t buf, int which, int q4) __attribute__((always_inline)) {
    return *reinterpret_cast<const af4_t *>(&s_s[buf][which][8 * q4 + 4 * half_id]);
  };
  auto seen = [&](uint32_t kb, int r) __attribute__((always_inline)) { return kb + 8 * (r / 4) + 4 * half_id + r % 4 <= pos; };
  // Scores to exponents relative to m, which moves where they need it.
  auto refer = [&](uint32_t kb, uint32_t buf, auto is_masked) __attribute__((always_inline)) {
    constexpr bool masked = decltype(is_masked)::value;
    // The largest u + log2 b: key by key where some are not seen (those must
    // change nothing), else from the largest of both.
    float top = -INFINITY;
#pragma unroll
    for (int q4 = 0; q4 < 4; q4++) {
      af4_t a, b;
      if constexpr (QUANT) a = scales(buf, 0, q4);
      if constexpr (QUANT && masked) b = scales(buf, 1, q4);
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int r = 4 * q4 + i;
        u[r] = QUANT ? fmaf(u[r], a[i], -m) : u[r] - m;
        if constexpr (masked) u[r] = seen(kb, r) ? u[r] : -INFINITY;
        top = fmaxf(top, QUANT && masked ? u[r] + scale_log(b[i]) : u[r]);
      }
    }
    if constexpr (QUANT) top += masked ? -127.f : fmaxf(top_s[buf][0], top_s[buf][1]);
    if (__builtin_amdgcn_ballot_w64(top > lazy)) {
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const bool move = top > lazy;  // the same in both lanes of a row
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
    }
  };
  ah8_t ph[2], pl[2];
  auto probabilities = [&](uint32_t kb, uint32_t buf, auto is_masked) __attribute__((always_inline)) {
    constexpr bool masked = decltype(is_masked)::value;
#pragma unroll
    for (int q4 = 0; q4 < 4; q4++) {
      af4_t b;
      if constexpr (QUANT) b = scales(buf, 1, q4);
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        const int r = 4 * q4 + i;
        const float p0 = __builtin_amdgcn_exp2f(u[r]), p1 = __builtin_amdgcn_exp2f(u[r + 1]);
        l += p0 + p1;
        af2_t pv = {p0, p1};
        if constexpr (QUANT) {
          // (A scale may be NaN, which 0 times it would be too.)
          if constexpr (masked) b[i] = seen(kb, r) ? b[i] : 0.f, b[i + 1] = seen(kb, r + 1) ? b[i + 1] : 0.f;
          pv = {p0 * b[i], p1 * b[i + 1]};
        }
        const ah2_t h = __builtin_convertvector(pv, ah2_t);
        const af2_t rest = {pv[0] - (float)h[0], pv[1] - (float)h[1]};
        const ah2_t e = __builtin_convertvector(rest, ah2_t);
        ph[r / 8][r % 8] = h[0], ph[r / 8][r % 8 + 1] = h[1];
        pl[r / 8][r % 8] = e[0], pl[r / 8][r % 8 + 1] = e[1];
      }
    }
  };
  auto value = [&](uint32_t buf, int j, uint32_t b) __attribute__((always_inline)) {
    return *reinterpret_cast<const ah8_t *>(&v_s[buf][((2 * j + half_id) * HD + 32 * b + col) * 8]);
  };
  // O^T += V^T·P^T.
  auto add = [&](ah8_t a, int j, uint32_t b) __attribute__((always_inline)) {
    o[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, ph[j], o[b], 0, 0, 0);
    o[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, pl[j], o[b], 0, 0, 0);
  };

  stage_keys(it.lo & 1);
  look_up(it.lo + 1);
  load_values(it.lo);
  load_keys(it.lo + 1);
  const bool plain = !__syncthreads_or(far || !active);
  u = scores(it.lo & 1);
  stage_keys(~it.lo & 1);
  stage_values(it.lo & 1, 32 * it.lo, std::true_type{});
  look_up(it.lo + 2);
  load_values(it.lo + 1);
  load_keys(it.lo + 2);
  look_up(it.lo + 3);
  lds_barrier();
  // Now, for step t: u its products; the keys of t + 1 and the values of t in
  // LDS; the keys of t + 2 and the values of t + 1 on their way to registers.
  uint32_t t = it.lo;
  if (plain) {
    // Steps that every row sees whole, the next one too.
    for (; t < last_step && 32 * t + 63 <= wg_pos0; t++) {
      const uint32_t now = t & 1, then = ~t & 1;
      refer(32 * t, now, std::false_type{});
      const af16_t next = scores(then);
      probabilities(32 * t, now, std::false_type{});
#pragma unroll
      for (int j = 0; j < 2; j++)
#pragma unroll
        for (uint32_t b = 0; b < OB; b++) add(value(now, j, b), j, b);
      stage_keys(now);
      stage_values(then, 32 * (t + 1), std::false_type{});
      load_values(t + 2);
      load_keys(t + 3);
      look_up(t + 4);
      u = next;
      lds_barrier();
    }
  }
  // The others.
  for (; t <= last_step; t++) {
    const uint32_t kb = 32 * t, now = t & 1, then = ~t & 1;
    if (active && kb < kend) {
      if (far) {
#pragma unroll
        for (int r = 0; r < 16; r++) u[r] *= back;
      }
      refer(kb, now, std::true_type{});
      probabilities(kb, now, std::true_type{});
      if (t < last_step) u = scores(then);
      const bool odd = !QUANT && (odd_s[now][0] | odd_s[now][1] | odd_s[now][2] | odd_s[now][3]);
#pragma unroll
      for (int j = 0; j < 2; j++)
#pragma unroll
        for (uint32_t b = 0; b < OB; b++) {
          ah8_t a = value(now, j, b);
          if constexpr (!QUANT) {
            // 0 times a value that is not finite is NaN: rows that see such a
            // value get it from a count, and the product leaves it out.
            if (odd) {
              ah8_t sees, bad;
              af16_t count;
#pragma unroll
              for (int i = 0; i < 16; i++) count[i] = 0.f;
#pragma unroll
              for (int i = 0; i < 8; i++) {
                sees[i] = (_Float16)(kb + 16 * j + 4 * half_id + (i & 4) * 2 + (i & 3) <= pos ? 1.f : 0.f);
                bad[i] = (_Float16)(not_finite(a[i]) ? 1.f : 0.f);
                a[i] = not_finite(a[i]) ? (_Float16)0.f : a[i];
              }
              count = __builtin_amdgcn_mfma_f32_32x32x16_f16(bad, sees, count, 0, 0, 0);
#pragma unroll
              for (int i = 0; i < 16; i++) o[b][i] = count[i] > 0.f ? NAN : o[b][i];
            }
          }
          add(a, j, b);
        }
    }
    stage_keys(now);
    stage_values(then, 32 * (t + 1), std::true_type{});
    load_values(t + 2);
    load_keys(t + 3);
    look_up(t + 4);
    lds_barrier();
  }
  // (Every wave has passed the last step's barrier: the next item may write to
  // the buffers.)
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
// parts-th of a row's records each, eight in flight, and meet in LDS.
template <uint32_t HD>
__global__ __launch_bounds__(256) void k_attn_join(const KvJoinItem *__restrict__ items, uint32_t n_kv, uint32_t group,
                                                   uint32_t parts, AttnOut to) {
  constexpr uint32_t N = 8, WIDE = HD / 4, GROUPS = 256 / WIDE;
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

// Deals the tiles' steps to at most `most` workgroups for each KV head in equal
// shares, cutting a tile where a share ends: all workgroups run at once and end
// together, and a tile is cut no more often than that takes.  A piece costs
// kStart steps besides its own (its queries, its results) and has `least` at
// least; with `whole` no tile is cut.  Tiles whose pieces' records have no room
// stay whole.
static void deal(KvSchedule &w, KvWork &work, std::vector<Tile> &tiles, uint64_t most, uint32_t least, bool whole,
                 uint32_t n_kv, uint64_t records) {
  constexpr uint64_t kStart = 4;
  work.starts.push_back(0);
  if (tiles.empty()) return;
  uint64_t total = 0;
  for (const Tile &t : tiles) total += t.steps + kStart;
  most = std::max<uint64_t>(most, 1);
  uint64_t groups = whole ? std::min<uint64_t>(most, tiles.size()) : std::min(most, std::max<uint64_t>(total / (least + kStart), 1));
  const uint64_t share = std::max<uint64_t>((total + kStart * groups + groups - 1) / groups, least + kStart);
  uint64_t room = share, dealt = 1;  // of the open workgroup; workgroups opened
  auto close = [&]() {
    if (work.starts.back() == work.items.size() || dealt == groups) return;
    work.starts.push_back((uint32_t)work.items.size());
    room = share;
    dealt++;
  };
  for (Tile &t : tiles) {
    const uint64_t rows = (uint64_t)n_kv * t.it.rows;
    const size_t first = work.items.size();
    for (uint32_t at = 0; at < t.steps;) {
      const uint32_t left = t.steps - at;
      // No room for a piece: the next workgroup's.
      if (room < left + kStart && (whole || room < least + kStart)) close();
      uint32_t take = left;
      if (!whole && dealt < groups && room < left + kStart && left >= 2 * least && w.records + 2 * rows <= records) {
        take = std::max((uint32_t)(room > kStart ? room - kStart : 0), least);
        take = std::min(take, left - least);
      }
      t.it.lo = at;
      t.it.hi = at + take;
      t.it.part = (uint32_t)w.records;
      if (take < t.steps) w.records += rows;
      work.items.push_back(t.it);
      at += take;
      room -= std::min<uint64_t>(room, take + kStart);
    }
    const uint32_t pieces = (uint32_t)(work.items.size() - first);
    if (pieces == 1)
      work.items[first].part = ~0u;
    else
      w.join.push_back({t.it.row, t.it.first, t.it.rows, pieces, work.items[first].part});
  }
  work.starts.push_back((uint32_t)work.items.size());
}

KvSchedule kv_schedule(const std::vector<KvSeq> &seqs, uint32_t group, uint32_t n_kv, uint32_t format, uint32_t head_dim,
                       uint32_t n_cus, uint64_t partial_floats) {
  KvSchedule w;
  const uint64_t records = std::min<uint64_t>(partial_floats / (head_dim + 4), 0xfffffffeu);
  if (!n_cus) n_cus = 256;
  // Which tiles.  Up to 32 rows take narrow tiles, which read the keys again
  // for every 16 rows (twelve sequences of about 2,000 keys, 20 and 32 rows,
  // heads of 64: 23 and 24 us against 26 and 26 in wide ones; of 256: 27 and 37
  // against 44 and 46).  Up to 128 rows do while the batch is small, because a
  // wide tile's few waves then wait for one another (1,000 keys, 96 rows, heads
  // of 128: 11 us against 20; at ten times the keys they are level).
  constexpr uint32_t kFewRows = 32;
  constexpr uint64_t kSmallBatch = 1u << 20;  // narrow tiles x steps x KV heads x head_dim
  uint64_t narrow_work = 0;
  for (const KvSeq &q : seqs) {
    const uint64_t rows = (uint64_t)q.n_new * group;
    if (rows > 16 && rows <= kChunkRows) narrow_work += (rows + 15) / 16 * ((q.past + q.n_new + 31) / 32) * n_kv * head_dim;
  }
  const uint32_t few_rows = narrow_work <= kSmallBatch ? kChunkRows : kFewRows;
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
  if (narrow_steps < token_steps) {
    tokens.insert(tokens.end(), narrow.begin(), narrow.end());
    narrow.clear();
  }
  // Narrow tiles: pieces of eight steps (two a wave) are as short as pays, and
  // a join (about 2.5 us) pays from 24 steps on with heads of 64, 19 of 128, 16
  // of 256 (300 keys of 64: 5.6 us whole, 7.6 cut; 2,000: 14.2 and 9.0).
  const uint32_t unsplit = 14 + 640 / head_dim;
  const uint64_t few_groups = (uint64_t)n_cus * token_groups(format, head_dim) / n_kv;
  deal(w, w.tiles8, narrow, few_groups, 8, longest <= unsplit, n_kv, records);
  deal(w, w.tiles16, tokens, few_groups, 8, longest <= unsplit, n_kv, records);
  deal(w, w.chunks, chunks, (uint64_t)n_cus * chunk_groups(head_dim) / n_kv, 8, false, n_kv, records);
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
