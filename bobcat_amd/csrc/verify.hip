// Which drafted tokens stay, and the token after them: speculative sampling on
// trees.
//
// At a token with the target's probabilities p, and q that its children were drawn
// from, child x with uniform u stays if u·q(x) < p(x); else p becomes (p - q)+,
// normalised, and the next child is looked at.  After m rejections that is
//   (p - c_m·q)+ / S_m,  S_m = Σ (p - c_m·q)+,  c_0 = 0,  S_0 = 1,
//   c_{m+1} = c_m + S_m / (1 - Q_m),
// Q_m the draft's mass of the rejected children where they were drawn without
// replacement, else 0: ((p - cq)+/S - q/(1-Q))+ = (p - (c + S/(1-Q))·q)+ / S, and a
// rejected token, of which less was left than q/(1-Q), has 0 from then on.  So two
// numbers stand for what is left of p, and a rejection costs one sum over the
// vocabulary.  For children chosen without chance (q is 1 for each in its turn) what is left
// is p without them, and a rejection costs nothing.
//
//   k_verify_rows reads every token's logits once, in pieces of the vocabulary: the
//     largest, the first place of it, and the sum of the exponentials.  Bound by
//     those bytes: 231 rows of 151,936 logits 26 us (5.4 TB/s, some of it out of the caches); with
//     f32 sums, which lose what is below 2^-24 of a thread's or a wave's, 24.6.
//   k_verify_walk walks down each tree, out of LDS, and draws: the piece in which the sum passes
//     its goal, then the token in it.  Without a draft a workgroup does a sequence.  With one
//     (REST) a workgroup for each piece walks by itself to where the sum for a rejection is missing,
//     adds its own piece to it, and the last one to do so goes on.  (One workgroup's sum
//     over 151,936 logits takes about 50 us.)  For trees there are launches before it that only add pieces,
//     for the first rejections; what those do not cover the last workgroup sums alone.  Bound by latency, some
//     fifteen loads that wait for each other, and code that runs once: one sequence of 5 tokens 12 us, 48 of up to 6
//     16 us.  (So lanes are summed by row moves, not through LDS, and a piece's elements have no branches: 14.5 and 19.2.)
#include <algorithm>
#include <cmath>

#include "device.h"
#include "kernels.h"
#include "kv_cache.h"
#include "runtime.h"

namespace bch {

constexpr uint32_t kRowThreads = 256, kRowPer = 16, kPiece = kRowThreads * kRowPer;
constexpr uint32_t kWalkThreads = 256;
// Rejections of trees that all workgroups sum, a launch each (of chains there is one at most).  Passes with
// 0, 1, 2, 3, 4, 5 and 6 of them: 16 trees of 16 to 32 drawn drafts, 65,536 logits, 101, 82, 74, 66, 62, 65 and
// 71 us; 8 of 8 to 16, without replacement, 151,936 logits, 153, 100, 77, 59, 47, 53 and 58; one of 16 drawn ones
// 51, 42, 33, 32, 34, 39 and 45.  (With f32 sums within a piece; f64 ones take about 1 us more of each pass.)
constexpr uint32_t kRounds = 4;
constexpr float kLargest = 3.402823466e38f;

// One piece of a row: its largest logit, where it is first, and the sum of
// exp((x - largest) / temperature).
struct VerifyPiece {
  double sum;
  float top;
  uint32_t at;
};

struct VerifyArgs {
  const float *logits, *draft;  // draft may be null
  const uint32_t *tokens;
  const float *uniforms, *temperatures;
  uint32_t *kept, *path, *next;
  float *chances;               // or null
  const KvSeq *seqs;            // of the first sequence on
  const KvNode *nodes;          // from the first token on, or null: chains
  VerifyPiece *pieces;          // [row][piece]
  double *rest;                 // [round][sequence][piece], one round more than `rounds`
  uint32_t *arrived;            // [sequence]
  uint32_t n_seqs, row0, n_rows, n_vocab, n_pieces, distinct;
  uint32_t rounds, most;        // rejections that are summed by all workgroups; the most tokens of a sequence
};

// A logit as it counts: NaN as -inf, +inf as the largest float.
__device__ __forceinline__ float logit(float x) { return x == x ? fminf(x, kLargest) : -INFINITY; }

// log2 e / temperature in two floats, so that x·(hi + lo) is off by its own rounding
// alone; kept off 0 and inf, which would make NaN of 0·inf.
struct Heat {
  float hi, lo, far;
  __device__ explicit Heat(float temperature) {
    const double c = fmin(fmax(1.44269504088896340736 / (double)temperature, 1e-30), 3e38);
    hi = (float)c;
    lo = (float)(c - (double)hi);
    far = -256.f / hi;  // (from there on the weight is 0)
  }
  // exp((x - top) / temperature) of a logit that is no larger than `top`.
  __device__ __forceinline__ float weight(float x, float top) const {
    const float d = x - top;
    return __builtin_amdgcn_exp2f(fmaf(d, hi, fmaxf(d, far) * lo));
  }
};

// What DPP control CTRL names, for the rows of 16 lanes of ROWS; 0 where there is none.
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ uint32_t dpp_u32(uint32_t x) {
  return __builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ double dpp_f64(double x) {
  const uint64_t v = __builtin_bit_cast(uint64_t, x);
  return __builtin_bit_cast(double, (uint64_t)dpp_u32<CTRL, ROWS>(v >> 32) << 32 | dpp_u32<CTRL, ROWS>((uint32_t)v));
}
// The sum of the lanes up to and with this one: within rows of 16 (from 1, 2, 4 and 8 lanes before), then the first and third
// rows' into the second and fourth, then the first half's into the second.
__device__ __forceinline__ double wave_scan_f64(double x) {
  x += dpp_f64<0x111>(x);
  x += dpp_f64<0x112>(x);
  x += dpp_f64<0x114>(x);
  x += dpp_f64<0x118>(x);
  x += dpp_f64<0x142, 0xa>(x);
  x += dpp_f64<0x143, 0xc>(x);
  return x;
}
// Lane `from`'s, the same for the wave.
__device__ __forceinline__ double lane_f64(double x, uint32_t from) {
  const uint64_t v = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)v, from), hi = __builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), from);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double wave_sum_f64(double x) { return lane_f64(wave_scan_f64(x), 63); }
__device__ __forceinline__ uint32_t wave_min_u32(uint32_t x) {
#pragma unroll
  for (int i = 1; i < 64; i *= 2) x = min(x, (uint32_t)__shfl_xor((int)x, i, 64));
  return x;
}

// The sequence of a row (rows of a sequence are consecutive): the last that
// begins at or before it, 64 at a time.
__device__ __forceinline__ uint32_t seq_of_row(const VerifyArgs &a, uint32_t row) {
  uint32_t lo = 0, count = a.n_seqs;
  while (count > 1) {
    const uint32_t step = (count + 63) / 64, i = threadIdx.x % 64 * step;
    const bool before = i < count && a.seqs[lo + min(i, count - 1)].row - a.row0 <= row;
    const uint32_t n = __popcll(__builtin_amdgcn_ballot_w64(before));
    lo += (n - 1) * step;
    count = min(step, count - (n - 1) * step);
  }
  return lo;
}

// VEC: rows are 16-byte aligned.
template <bool VEC>
__global__ __launch_bounds__(kRowThreads) void k_verify_rows(VerifyArgs a) {
  __shared__ float top_s[4];
  __shared__ double sum_s[4];
  __shared__ uint32_t at_s[4];
  const uint32_t row = blockIdx.x / a.n_pieces, piece = blockIdx.x % a.n_pieces, tid = threadIdx.x;
  const uint32_t base = piece * kPiece, len = min(kPiece, a.n_vocab - base);
  const float *p = a.logits + (uint64_t)row * a.n_vocab + base;
  float x[kRowPer];
  // Element j of a thread is at place(j).
  auto place = [&](uint32_t j) { return VEC ? 4 * (tid + kRowThreads * (j / 4)) + j % 4 : tid + kRowThreads * j; };
  if constexpr (VEC) {
#pragma unroll
    for (uint32_t j = 0; j < kRowPer; j += 4) {
      const float4 v = *reinterpret_cast<const float4 *>(p + min(place(j), len - 4));
      x[j] = v.x, x[j + 1] = v.y, x[j + 2] = v.z, x[j + 3] = v.w;
    }
  } else {
#pragma unroll
    for (uint32_t j = 0; j < kRowPer; j++) x[j] = p[min(place(j), len - 1)];
  }
  const uint32_t seq = seq_of_row(a, row);
  const float temperature = a.temperatures[seq];
  if (piece == 0 && tid == 0 && a.seqs[seq].row - a.row0 == row) a.arrived[seq] = 0;
  float top = -INFINITY;
#pragma unroll
  for (uint32_t j = 0; j < kRowPer; j++) {
    x[j] = place(j) < len ? logit(x[j]) : -INFINITY;
    top = fmaxf(top, x[j]);
  }
  top = block_max<kRowThreads>(top, top_s);
  // The first place of the largest.
  uint32_t at = ~0u;
#pragma unroll
  for (int j = kRowPer - 1; j >= 0; j--)
    if (x[j] == top) at = base + place(j);
  at = wave_min_u32(at);
  double sum = 0;  // (of f32 terms, as every sum over the vocabulary here)
  if (temperature > 0.f && top > -INFINITY) {
    const Heat heat(temperature);
#pragma unroll
    for (uint32_t j = 0; j < kRowPer; j++) sum += (double)heat.weight(x[j], top);
  }
  sum = wave_sum_f64(sum);
  if (tid % 64 == 0) at_s[tid / 64] = at, sum_s[tid / 64] = sum;
  __syncthreads();
  if (tid == 0)
    a.pieces[blockIdx.x] = {(sum_s[0] + sum_s[1]) + (sum_s[2] + sum_s[3]), top, min(min(at_s[0], at_s[1]), min(at_s[2], at_s[3]))};
}

// What a workgroup knows of its sequence, in LDS: of each token its row's largest
// logit, sum and first largest's place, its own probabilities (after its parent), and the tree.
struct WalkMemory {
  double *sum, *p, *q;
  float *top, *u;
  uint32_t *best, *token, *child, *sibling, *path;
  __device__ WalkMemory(double *at, uint32_t n) {
    sum = at, p = sum + n, q = p + n;
    top = reinterpret_cast<float *>(q + n), u = top + n;
    best = reinterpret_cast<uint32_t *>(u + n), token = best + n, child = token + n, sibling = child + n, path = sibling + n;
  }
};
constexpr uint32_t kWalkBytes = 3 * 8 + 7 * 4;  // a token

struct Walk {
  const VerifyArgs &a;
  const uint32_t seq_at;
  const KvSeq seq;
  const uint32_t n, row0;
  const float temperature;
  const bool greedy, drawn;
  const Heat heat;
  const double heat64;
  WalkMemory m;
  // The current token and the kept ones, and what is left of p: (p - c·q)+ with the sum of `round`.
  uint32_t t = 0, kept = 1, round = 0;
  double c = 0;

  __device__ Walk(const VerifyArgs &args, uint32_t which, double *memory)
      : a(args), seq_at(which), seq(args.seqs[which]), n(seq.n_new), row0(seq.row - args.row0),
        temperature(args.temperatures[which]), greedy(!(temperature > 0.f)), drawn(args.draft && !greedy),
        heat(greedy ? 1.f : temperature), heat64((double)heat.hi + (double)heat.lo), m(memory, args.most) {}

  // The target's probability of token x after token i.
  __device__ double chance(uint32_t i, uint32_t x) const {
    if (x >= a.n_vocab || m.best[i] == BCH_NO_TOKEN) return 0.0;
    if (greedy) return x == m.best[i] ? 1.0 : 0.0;
    const float l = logit(a.logits[(uint64_t)(row0 + i) * a.n_vocab + x]);
    return l > -INFINITY ? exp2(((double)l - m.top[i]) * heat64) / m.sum[i] : 0.0;
  }

  // The rows' pieces joined, 16 lanes a row, and every drafted token's probabilities.
  __device__ void load(bool chances) {
    const uint32_t tid = threadIdx.x, lane = tid % 16;
    const KvNode *nodes = a.nodes ? a.nodes + row0 : nullptr;
    for (uint32_t i = tid; i < n; i += kWalkThreads) {
      m.token[i] = a.tokens[row0 + i];
      m.u[i] = a.uniforms[row0 + i];
      m.child[i] = nodes ? nodes[i].child : i + 1 < n ? i + 1 : kKvNone;
      m.sibling[i] = nodes ? nodes[i].sibling : kKvNone;
      m.path[i] = nodes ? nodes[i].parent : i - 1;  // (until the probabilities are known)
    }
    for (uint32_t i0 = 0; i0 < n; i0 += kWalkThreads / 16) {
      const uint32_t i = min(i0 + tid / 16, n - 1);
      const VerifyPiece *p = a.pieces + (uint64_t)(row0 + i) * a.n_pieces;
      // (A running sum: rows of up to 64 pieces, 262,144 tokens, in one round of loads.)
      float top = -INFINITY;
      double sum = 0;
      uint32_t best = ~0u;
#pragma unroll 1
      for (uint32_t j0 = 0; j0 < a.n_pieces; j0 += 64) {
        VerifyPiece x[4];
#pragma unroll
        for (uint32_t k = 0; k < 4; k++) x[k] = p[min(j0 + 16 * k + lane, a.n_pieces - 1)];
        const float before = top;
#pragma unroll
        for (uint32_t k = 0; k < 4; k++) {
          if (j0 + 16 * k + lane >= a.n_pieces) x[k] = {0, -INFINITY, ~0u};
          best = x[k].top > top ? x[k].at : best;  // (pieces go up, and so do the places)
          top = fmaxf(top, x[k].top);
        }
        if (before > -INFINITY) sum *= heat.weight(before, top);
#pragma unroll
        for (uint32_t k = 0; k < 4; k++)
          if (x[k].top > -INFINITY) sum += x[k].sum * heat.weight(x[k].top, top);
      }
      float all = fmaxf(top, dpp<kDppXor1>(top));
      all = fmaxf(all, dpp<kDppXor2>(all));
      all = fmaxf(all, dpp<kDppHalfMirror>(all));
      all = fmaxf(all, dpp<kDppMirror>(all));
      if (top > -INFINITY) sum *= heat.weight(top, all);
      if (top != all) best = ~0u;
      sum += dpp_f64<kDppXor1>(sum);
      sum += dpp_f64<kDppXor2>(sum);
      sum += dpp_f64<kDppHalfMirror>(sum);
      sum += dpp_f64<kDppMirror>(sum);
      best = min(best, dpp_u32<kDppXor1>(best));
      best = min(best, dpp_u32<kDppXor2>(best));
      best = min(best, dpp_u32<kDppHalfMirror>(best));
      best = min(best, dpp_u32<kDppMirror>(best));
      if (lane == 0) m.top[i] = all, m.sum[i] = sum, m.best[i] = all > -INFINITY ? best : BCH_NO_TOKEN;
    }
    __syncthreads();
    for (uint32_t i = tid; i < n; i += kWalkThreads) {
      if (!i) {
        m.path[0] = 0;
        continue;
      }
      const uint32_t up = m.path[i], x = m.token[i];
      const double p = chance(up, x);
      // (Children chosen without chance that name a token again find nothing left of it.)
      bool again = false;
      if (!drawn)
        for (uint32_t s = m.child[up]; s != i; s = m.sibling[s]) again |= m.token[s] == x;
      m.p[i] = again ? 0.0 : p;
      m.q[i] = !drawn ? 1.0 : x < a.n_vocab ? (double)a.draft[(uint64_t)(row0 + up) * a.n_vocab + x] : 0.0;
      m.path[i] = BCH_NO_TOKEN;
      if (chances) a.chances[row0 + i] = (float)p;
    }
    __syncthreads();
  }

  // Down the tree, from its first token or from where it stopped; total_of(round) is the sum of
  // (p - c·q)+, or below 0 where it is not known yet: false then.
  uint32_t looked = kKvNone;  // the child whose rejection waits for its sum
  double left = 1, total = 1;
  template <class Total>
  __device__ bool down(Total &&total_of) {
    for (;;) {
      uint32_t s = looked;
      if (s == kKvNone) {
        c = 0, left = total = 1;
        s = m.child[t];
      }
      for (; s != kKvNone; s = m.sibling[s]) {
        const double u = (double)m.u[s], p = m.p[s], q = m.q[s];
        if (looked == kKvNone) {
          // (A child's q is part of the draft's mass that is left, but for roundings of the f32 probabilities.)
          if (a.distinct) left = fmax(left, q);
          if (p > 0 && (greedy ? true : drawn ? p > c * q && u * q * total < (p - c * q) * left : u * total < p)) break;
          if (drawn) {
            if (left > 0) c += total / left;
            if (a.distinct) left -= q;
          } else if (!greedy) {
            total -= p;
          }
        }
        if (drawn) {
          looked = s;
          const double sum = total_of(round);
          if (sum < 0) return false;
          total = sum;
          looked = kKvNone;
          round++;
        }
      }
      if (s == kKvNone) return true;
      if (threadIdx.x == 0) m.path[kept] = s;
      kept++;
      t = s;
    }
  }

  // A piece of (p - c·q)+ after the current token, or of p in units of its largest; 0 behind the vocabulary.
  struct Piece {
    const float *logits, *draft;
    float top, inv, c;
    uint32_t len;
    // Elements `first` + STRIDE·j of it, all on their way before one is used.  (Buffer loads end at the
    // piece by themselves: clamped places would take a register each.)
    template <uint32_t STRIDE, uint32_t N>
    __device__ __forceinline__ void load(const Heat &heat, float (&x)[N], uint32_t first) const {
      float d[N] = {};
      auto bring = [&](float (&to)[N], const float *from) __attribute__((always_inline)) {
        const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(from), 0, len * 4, 0x00020000);
#pragma unroll
        for (uint32_t j = 0; j < N; j++)
          to[j] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rsrc, 4 * first, 4 * STRIDE * j, 0));
      };
      bring(x, logits);
      if (draft) bring(d, draft);
#pragma unroll
      for (uint32_t j = 0; j < N; j++) {
        const float p = heat.weight(first + STRIDE * j < len ? logit(x[j]) : -INFINITY, top) * inv;
        // (What the target does not have stays at 0, whatever the draft says.  Without a draft c is 0.)
        x[j] = p > 0.f ? fmaxf(fmaf(-c, d[j], p), 0.f) : 0.f;
      }
    }
  };
  __device__ Piece piece_of(uint32_t piece) const {  // (the same for a wave)
    const uint32_t at_t = __builtin_amdgcn_readfirstlane(t), from = __builtin_amdgcn_readfirstlane(piece) * kPiece;
    const uint64_t at = (uint64_t)(row0 + at_t) * a.n_vocab + from;
    return {a.logits + at, c > 0 ? a.draft + at : nullptr, fmaxf(m.top[t], -kLargest), c > 0 ? (float)(1.0 / m.sum[t]) : 1.f,
            c > 0 ? (float)c : 0.f, min(kPiece, a.n_vocab - from)};
  }
  __device__ double *rest(uint32_t which) const { return a.rest + ((uint64_t)which * a.n_seqs + seq_at) * a.n_pieces; }
  // The sum of a round's pieces (never below 0), by each wave for itself.
  double held = 0;  // of up to 64 pieces this lane's of the last round
  __device__ double total_of_pieces(uint32_t which) {
    const double *p = rest(which);
    double sum = 0;
    for (uint32_t i = threadIdx.x % 64; i < a.n_pieces; i += 64) sum += coherent_load(p + i);
    held = sum;
    return wave_sum_f64(sum);
  }
  // A wave's sum of a piece of it.
  __device__ double piece_by_wave(uint32_t piece) const {
    const Piece part = piece_of(piece);
    double sum = 0;
#pragma unroll 1
    for (uint32_t j0 = 0; j0 < kPiece / 64; j0 += 8) {
      float x[8];
      part.load<64>(heat, x, 64 * j0 + threadIdx.x % 64);
#pragma unroll
      for (uint32_t j = 0; j < 8; j++) sum += (double)x[j];
    }
    return wave_sum_f64(sum);
  }

  // The next token; `latest` is the round of the last c.
  __device__ uint32_t next(uint32_t latest) {
    constexpr uint32_t WAVES = kWalkThreads / 64, PER = kPiece / kWalkThreads;
    __shared__ double run_s[WAVES];
    __shared__ uint32_t pick_s[WAVES], last_s[WAVES];
    __shared__ float x_s[kWalkThreads * (PER + 1)];  // (a place in 17 is free: no bank is met twice)
    const uint32_t tid = threadIdx.x, wave = tid / 64, lane = tid % 64;
    if (greedy || m.best[t] == BCH_NO_TOKEN) return m.best[t];
    bool without = !drawn && m.child[t] != kKvNone;  // without the children that were chosen
    auto mass = [&](uint32_t piece) {
      if (c > 0) return a.n_pieces <= 64 ? held : coherent_load(rest(latest) + piece);
      const VerifyPiece p = a.pieces[(uint64_t)(row0 + t) * a.n_pieces + piece];
      double sum = p.top > -INFINITY ? p.sum * heat.weight(p.top, m.top[t]) : 0.0;
      if (without)
        for (uint32_t s = m.child[t]; s != kKvNone; s = m.sibling[s])
          if (m.token[s] / kPiece == piece) sum -= m.p[s] * m.sum[t];
      return fmax(sum, 0.0);
    };
    // Every wave finds the piece for itself, a lane has `per` consecutive ones.
    const uint32_t per = (a.n_pieces + 63) / 64, first = min(lane * per, a.n_pieces), end = min(first + per, a.n_pieces);
    for (;; c = 0, without = false) {  // (where nothing is left: p itself)
      double mine = 0;
      for (uint32_t i = first; i < end; i++) mine += mass(i);
      const double up = wave_scan_f64(mine), total = lane_f64(up, 63);
      const bool itself = c == 0 && !without;
      if (!(total > 0) && !itself) continue;
      // The first piece whose end lies past the goal; the last with any mass where rounding leaves none.
      const double goal = (double)m.u[0] * total;
      const uint64_t past = __builtin_amdgcn_ballot_w64(mine > 0 && up > goal), any = __builtin_amdgcn_ballot_w64(mine > 0);
      const bool inside = past != 0;
      const uint32_t owner = inside ? __ffsll((unsigned long long)past) - 1 : any ? 63 - __clzll((long long)any) : 0;
      double sum = up - mine;
      uint32_t from = first;
      if (per > 1) {
        double at = sum;
        bool passed = false;
        for (uint32_t i = first; i < end; i++) {
          const double x = mass(i);
          if (x > 0 && !passed) from = i, sum = at, passed = inside && at + x > goal;
          at += x;
        }
      }
      sum = lane_f64(sum, __builtin_amdgcn_readfirstlane(owner));
      from = __builtin_amdgcn_readlane((int)from, __builtin_amdgcn_readfirstlane(owner));
      // The token in the piece.  Its own sum may end below the goal by rounding: the last token with any weight
      // then, or where it has none (all of it was fallen children) the pieces behind it, then those before.
#pragma unroll 1
      for (uint32_t k = 0; k < a.n_pieces; k++) {
        const uint32_t piece = from + k < a.n_pieces ? from + k : a.n_pieces - 1 - k;
        // Read side by side, and taken PER in a row.  (Eight at a time, for the registers.)
        {
          const Piece part = piece_of(piece);
#pragma unroll 1
          for (uint32_t i0 = tid; i0 < kPiece; i0 += kWalkThreads * 8) {
            float x[8];
            part.load<kWalkThreads>(heat, x, i0);
#pragma unroll
            for (uint32_t j = 0; j < 8; j++) {
              const uint32_t i = i0 + kWalkThreads * j;
              x_s[i + i / PER] = x[j];
            }
          }
        }
        __syncthreads();
        if (without) {
          for (uint32_t s = m.child[t]; s != kKvNone; s = m.sibling[s]) {
            const uint32_t i = m.token[s] - piece * kPiece;
            if (i < kPiece) x_s[i + i / PER] = 0.f;  // (every thread the same)
          }
          __syncthreads();
        }
        const float *mine_s = x_s + tid * (PER + 1);
        double run = 0;
#pragma unroll 4
        for (uint32_t j = 0; j < PER; j++) run += (double)mine_s[j];
        const double upto = wave_scan_f64(run);
        if (lane == 63) run_s[wave] = upto;
        __syncthreads();
        double at = sum + upto - run;
        for (uint32_t i = 0; i < wave; i++) at += run_s[i];
        uint32_t pick = ~0u, last = ~0u;  // (places go up with the lanes)
#pragma unroll 4
        for (uint32_t j = 0; j < PER; j++) {
          const float x = mine_s[j];
          at += (double)x;
          const uint32_t i = piece * kPiece + PER * tid + j;
          if (x > 0.f) last = i;
          if (x > 0.f && pick == ~0u && at > goal && inside) pick = i;
        }
        const uint64_t picks = __builtin_amdgcn_ballot_w64(pick != ~0u), lasts = __builtin_amdgcn_ballot_w64(last != ~0u);
        if (picks ? lane == __ffsll((unsigned long long)picks) - 1 : lane == 0) pick_s[wave] = pick;
        if (lasts ? lane == 63 - __clzll((long long)lasts) : lane == 0) last_s[wave] = last;
        __syncthreads();
        for (uint32_t i = 0; i < WAVES; i++) {
          if (pick_s[i] != ~0u) return pick_s[i];
        }
        for (uint32_t i = WAVES; i-- > 0;) {
          if (last_s[i] != ~0u) return last_s[i];
        }
        __syncthreads();
      }
      // No token has any weight: what was left was roundings (a chosen child's p is f64, its term in a piece's sum
      // f32).  Of p itself the largest logit has the weight 1.
      if (itself) return BCH_NO_TOKEN;
    }
  }
};

// REST: workgroups for every piece of every sequence, of which those of the last launch also end the walk.
template <bool REST>
__global__ __launch_bounds__(kWalkThreads, REST ? 6 : 2) void k_verify_walk(VerifyArgs a, uint32_t known, bool last) {
  extern __shared__ double memory[];
  __shared__ double sum_s[kWalkThreads / 64];
  __shared__ uint32_t arrived_s;
  const uint32_t tid = threadIdx.x, wave = tid / 64, lane = tid % 64;
  const uint32_t piece = REST ? blockIdx.x % a.n_pieces : 0, which = REST ? blockIdx.x / a.n_pieces : blockIdx.x;
  Walk w(a, which, memory);
  if (REST && piece && !w.drawn) return;
  if (!w.n) {
    if (tid == 0 && last && !piece) a.kept[which] = 0, a.next[which] = BCH_NO_TOKEN;
    return;
  }
  w.load(a.chances && last && !piece);
  uint32_t latest = 0;  // the round whose pieces are those of the last c
  bool open = true;
  if (REST) {
    open = !w.down([&](uint32_t round) {
      latest = round;
      return round < known ? w.total_of_pieces(round) : -1.0;
    });
    if (open) {
      float x[kPiece / kWalkThreads];
      w.piece_of(piece).load<kWalkThreads>(w.heat, x, tid);
      double sum = 0;
#pragma unroll
      for (uint32_t j = 0; j < kPiece / kWalkThreads; j++) sum += (double)x[j];
      const double by_wave = wave_sum_f64(sum);
      if (lane == 0) sum_s[wave] = by_wave;
      __syncthreads();
      if (tid == 0) {
        coherent_store(w.rest(known) + piece, (sum_s[0] + sum_s[1]) + (sum_s[2] + sum_s[3]));
        if (last) {
          // The piece is complete before it is counted.
          __atomic_signal_fence(__ATOMIC_SEQ_CST);
          __builtin_amdgcn_s_waitcnt(0);
          __atomic_signal_fence(__ATOMIC_SEQ_CST);
          arrived_s = __hip_atomic_fetch_add(a.arrived + which, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
      }
      if (!last) return;
      __syncthreads();
      if (arrived_s != a.n_pieces - 1) return;
    } else if (!last || piece) {
      return;
    }
  }
  if (open) w.down([&](uint32_t round) {
    latest = min(round, a.rounds);
    if (round >= a.rounds) {  // further rejections: a wave sums every fourth piece
      __syncthreads();
      for (uint32_t i = wave; i < a.n_pieces; i += kWalkThreads / 64) {
        const double sum = w.piece_by_wave(i);
        if (lane == 0) coherent_store(w.rest(latest) + i, sum);
      }
      __builtin_amdgcn_s_waitcnt(0);
      __syncthreads();
    }
    return w.total_of_pieces(latest);
  });
  const uint32_t next = w.next(latest);
  __syncthreads();  // (the path is thread 0's)
  for (uint32_t i = tid; i < w.n; i += kWalkThreads) a.path[w.row0 + i] = w.m.path[i];
  if (tid == 0) {
    a.kept[which] = w.kept;
    a.next[which] = next;
    if (a.chances) a.chances[w.row0] = next == BCH_NO_TOKEN ? 0.f : (float)w.chance(w.t, next);
  }
}

}  // namespace bch

using namespace bch;

extern "C" int bch_verify_drafts(bch_ctx *ctx, const bch_kv_plan *plan, uint32_t first, uint32_t n_seqs, uint32_t n_vocab,
                                 const bch_drafts *drafts, const bch_verdict *verdict) {
  if (!drafts || !verdict) return fail(BCH_ERR_ARGUMENT, "verify_drafts: no drafts or no verdict");
  BCH_TRY(kv_plan_ready(ctx, "verify_drafts", plan));
  VerifyArgs a{};
  BCH_TRY(kv_plan_range("verify_drafts", plan, first, n_seqs, &a.row0, &a.n_rows));
  if (!n_vocab || n_vocab > 1u << 30) return fail(BCH_ERR_ARGUMENT, "verify_drafts: rows of %u logits", n_vocab);
  for (uint32_t i = first; i < first + n_seqs; i++) {
    if (plan->seqs[i].n_new > BCH_MAX_TREE)
      return fail(BCH_ERR_ARGUMENT, "verify_drafts: sequence %u has %u tokens, at most %u are wanted", i, plan->seqs[i].n_new,
                  BCH_MAX_TREE);
    if (!plan->rooted.empty() && !plan->rooted[i])
      return fail(BCH_ERR_ARGUMENT, "verify_drafts: the drafts of sequence %u do not all follow its first token", i);
  }
  a.n_seqs = n_seqs;
  a.n_vocab = n_vocab;
  a.n_pieces = div_ceil(n_vocab, kPiece);
  a.distinct = drafts->distinct != 0;
  if ((uint64_t)std::max(a.n_rows, n_seqs) * a.n_pieces >= 1u << 23) return fail(BCH_ERR_ARGUMENT, "verify_drafts: too many logits");
  const uint64_t rows = a.n_rows, bytes = rows * n_vocab * 4;
  BCH_TRY(view_ptr(ctx, "verify_drafts", drafts->logits, bytes, &a.logits));
  if (drafts->draft.buffer) BCH_TRY(view_ptr(ctx, "verify_drafts", drafts->draft, bytes, &a.draft));
  BCH_TRY(view_ptr(ctx, "verify_drafts", drafts->tokens, rows * 4, &a.tokens));
  BCH_TRY(view_ptr(ctx, "verify_drafts", drafts->uniforms, rows * 4, &a.uniforms));
  BCH_TRY(view_ptr(ctx, "verify_drafts", drafts->temperatures, (uint64_t)n_seqs * 4, &a.temperatures));
  BCH_TRY(view_ptr(ctx, "verify_drafts", verdict->kept, (uint64_t)n_seqs * 4, &a.kept));
  BCH_TRY(view_ptr(ctx, "verify_drafts", verdict->path, rows * 4, &a.path));
  BCH_TRY(view_ptr(ctx, "verify_drafts", verdict->next, (uint64_t)n_seqs * 4, &a.next));
  if (verdict->chances.buffer) BCH_TRY(view_ptr(ctx, "verify_drafts", verdict->chances, rows * 4, &a.chances));
  struct Part {
    const void *at;
    uint64_t bytes;
  };
  const Part in[] = {{a.logits, bytes}, {a.draft, a.draft ? bytes : 0}, {a.tokens, rows * 4}, {a.uniforms, rows * 4},
                     {a.temperatures, (uint64_t)n_seqs * 4}};
  const Part out[] = {{a.kept, (uint64_t)n_seqs * 4}, {a.path, rows * 4}, {a.next, (uint64_t)n_seqs * 4},
                      {a.chances, a.chances ? rows * 4 : 0}};
  for (const Part &o : out) {
    for (const Part &i : in)
      if (kv_overlap(o.at, o.bytes, i.at, i.bytes))
        return fail(BCH_ERR_ARGUMENT, "verify_drafts: the verdict lies over the drafts");
    for (const Part &other : out)
      if (&other != &o && kv_overlap(o.at, o.bytes, other.at, other.bytes))
        return fail(BCH_ERR_ARGUMENT, "verify_drafts: parts of the verdict lie over each other");
  }
  for (const Part &x : in)
    if (reinterpret_cast<uintptr_t>(x.at) % 4) return fail(BCH_ERR_ARGUMENT, "verify_drafts: operands must be 4-byte aligned");
  for (const Part &x : out)
    if (reinterpret_cast<uintptr_t>(x.at) % 4) return fail(BCH_ERR_ARGUMENT, "verify_drafts: operands must be 4-byte aligned");
  if (!ctx->recording && !ctx->capturing) return fail(BCH_ERR_NOT_RECORDING, "no recording is open");
  for (uint32_t i = first; i < first + n_seqs; i++) a.most = std::max(a.most, plan->seqs[i].n_new);
  a.rounds = !a.draft || a.most < 2 ? 0 : plan->d_nodes ? std::min(kRounds, a.most - 1) : 1;
  const uint64_t pieces = rows * a.n_pieces * sizeof(VerifyPiece), rest = (uint64_t)n_seqs * a.n_pieces * 8;
  void *scratch;
  BCH_TRY(ctx_scratch(ctx, pieces + (a.rounds + 1) * rest + n_seqs * 4ull + 16, &scratch));
  a.pieces = static_cast<VerifyPiece *>(scratch);
  a.rest = reinterpret_cast<double *>(static_cast<char *>(scratch) + pieces);
  a.arrived = reinterpret_cast<uint32_t *>(static_cast<char *>(scratch) + pieces + (a.rounds + 1) * rest);
  return launch(ctx, {"verify_drafts", a.n_rows, n_vocab, 0}, [&](hipStream_t st) {
    if (!n_seqs) return;
    kv_plan_use(ctx, plan);
    a.seqs = plan->d_seqs + first;
    a.nodes = plan->d_nodes ? plan->d_nodes + a.row0 : nullptr;
    const uint32_t memory = a.most * kWalkBytes;
    if (a.n_rows) {
      if (n_vocab % 4 == 0 && reinterpret_cast<uintptr_t>(a.logits) % 16 == 0)
        k_verify_rows<true><<<a.n_rows * a.n_pieces, kRowThreads, 0, st>>>(a);
      else
        k_verify_rows<false><<<a.n_rows * a.n_pieces, kRowThreads, 0, st>>>(a);
    }
    if (!a.rounds)
      k_verify_walk<false><<<n_seqs, kWalkThreads, memory, st>>>(a, 0, true);
    for (uint32_t i = 0; i < a.rounds; i++)
      k_verify_walk<true><<<n_seqs * a.n_pieces, kWalkThreads, memory, st>>>(a, i, i + 1 == a.rounds);
  });
}
