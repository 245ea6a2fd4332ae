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
// k_verify_rows reads every token's logits once: the largest, the first place of it,
// and the sum of the exponentials, for pieces of the vocabulary.  k_verify_walk has a workgroup
// for each sequence: it joins the pieces of its rows and takes the probabilities of all
// drafted tokens at once, walks down (every thread the same way, out of LDS), and
// draws.
#include <algorithm>
#include <cmath>

#include "device.h"
#include "kernels.h"
#include "kv_cache.h"
#include "runtime.h"

namespace bch {

constexpr uint32_t kRowThreads = 256, kRowPer = 16, kRowPiece = kRowThreads * kRowPer;
constexpr uint32_t kWalkThreads = 1024, kWalkWaves = kWalkThreads / 64;
constexpr float kLargest = 3.402823466e38f;

// One piece of a row: its largest logit, where it is first, and the sum of
// exp((x - largest) / temperature).
struct VerifyPiece {
  float top, sum;
  uint32_t at, pad;
};

struct VerifyArgs {
  const float *logits, *draft;  // draft may be null
  const uint32_t *tokens;
  const float *uniforms, *temperatures;
  uint32_t *kept, *path, *next;
  float *chances;               // or null
  const KvSeq *seqs;            // of the first sequence on
  const KvNode *nodes;          // from the first token on, or null: chains
  VerifyPiece *pieces;
  uint32_t n_seqs, row0, n_rows, n_vocab, n_pieces, distinct;
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

__device__ __forceinline__ double wave_sum_f64(double x) {
#pragma unroll
  for (int i = 1; i < 64; i *= 2) x += __shfl_xor(x, i, 64);
  return x;
}

// The sequence of a row (rows of a sequence are consecutive).
__device__ __forceinline__ uint32_t seq_of_row(const VerifyArgs &a, uint32_t row) {
  uint32_t lo = 0, hi = a.n_seqs;  // the last with a first row <= row that has rows
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) / 2;
    if (a.seqs[mid].row - a.row0 <= row) lo = mid; else hi = mid;
  }
  return lo;
}

__global__ __launch_bounds__(kRowThreads) void k_verify_rows(VerifyArgs a) {
  __shared__ float top_s[4], sum_s[4];
  __shared__ uint32_t at_s[4];
  const uint32_t row = blockIdx.x / a.n_pieces, piece = blockIdx.x % a.n_pieces, tid = threadIdx.x;
  const uint32_t base = piece * kRowPiece, len = min(kRowPiece, a.n_vocab - base);
  const float *p = a.logits + (uint64_t)row * a.n_vocab + base;
  float x[kRowPer];
#pragma unroll
  for (uint32_t j = 0; j < kRowPer; j++) {
    const uint32_t i = tid + kRowThreads * j;
    x[j] = i < len ? logit(p[i]) : -INFINITY;
  }
  const float temperature = a.temperatures[seq_of_row(a, row)];
  float top = -INFINITY;
#pragma unroll
  for (uint32_t j = 0; j < kRowPer; j++) top = fmaxf(top, x[j]);
  top = block_max<kRowThreads>(top, top_s);
  // The first place of the largest.
  uint32_t at = ~0u;
#pragma unroll
  for (int j = kRowPer - 1; j >= 0; j--)
    if (x[j] == top) at = base + tid + kRowThreads * j;
#pragma unroll
  for (int i = 1; i < 64; i *= 2) at = min(at, (uint32_t)__shfl_xor((int)at, i, 64));
  float sum = 0.f;
  if (temperature > 0.f && top > -INFINITY) {
    const Heat heat(temperature);
#pragma unroll
    for (uint32_t j = 0; j < kRowPer; j++) sum += heat.weight(x[j], top);
  }
  sum = block_sum<kRowThreads>(sum, sum_s);
  if (tid % 64 == 0) at_s[tid / 64] = at;
  __syncthreads();
  if (tid == 0) a.pieces[blockIdx.x] = {top, sum, min(min(at_s[0], at_s[1]), min(at_s[2], at_s[3])), 0};
}

__global__ __launch_bounds__(kWalkThreads) void k_verify_walk(VerifyArgs a) {
  __shared__ float top_s[BCH_MAX_TREE];                      // of each token's row
  __shared__ double sum_s[BCH_MAX_TREE];                     // its sum; greedy: unused
  __shared__ uint32_t best_s[BCH_MAX_TREE];                  // the first place of its largest
  __shared__ double p_s[BCH_MAX_TREE], q_s[BCH_MAX_TREE];    // of each drafted token after its parent
  __shared__ uint32_t token_s[BCH_MAX_TREE], path_s[BCH_MAX_TREE];
  __shared__ bool again_s[BCH_MAX_TREE];                     // a sibling before it is the same token
  __shared__ double span_s[kWalkThreads];
  __shared__ double part_s[kWalkWaves];
  __shared__ uint32_t next_s;
  const uint32_t tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64), lane = tid % 64;
  const KvSeq seq = a.seqs[blockIdx.x];
  const uint32_t n = seq.n_new, row0 = seq.row - a.row0;
  if (!n) {
    if (tid == 0) a.kept[blockIdx.x] = 0, a.next[blockIdx.x] = BCH_NO_TOKEN;
    return;
  }
  const float temperature = a.temperatures[blockIdx.x];
  const bool greedy = !(temperature > 0.f), drawn = a.draft && !greedy;
  const Heat heat(greedy ? 1.f : temperature);
  const double heat64 = (double)heat.hi + (double)heat.lo;
  const KvNode *nodes = a.nodes ? a.nodes + row0 : nullptr;
  auto parent_of = [&](uint32_t t) { return nodes ? nodes[t].parent : t - 1; };
  auto child_of = [&](uint32_t t) { return nodes ? nodes[t].child : t + 1 < n ? t + 1 : kKvNone; };
  auto sibling_of = [&](uint32_t t) { return nodes ? nodes[t].sibling : kKvNone; };

  // The rows' pieces joined, a wave a row.
  for (uint32_t t = wave; t < n; t += kWalkWaves) {
    const VerifyPiece *p = a.pieces + (uint64_t)(row0 + t) * a.n_pieces;
    float top = -INFINITY;
    for (uint32_t i = lane; i < a.n_pieces; i += 64) top = fmaxf(top, p[i].top);
    top = wave_max(top);
    uint32_t best = ~0u;
    double sum = 0;
    for (uint32_t i = lane; i < a.n_pieces; i += 64) {
      if (p[i].top == top) best = min(best, p[i].at);
      if (p[i].top > -INFINITY) sum += (double)p[i].sum * exp2(((double)p[i].top - top) * heat64);
    }
#pragma unroll
    for (int i = 1; i < 64; i *= 2) best = min(best, (uint32_t)__shfl_xor((int)best, i, 64));
    sum = wave_sum_f64(sum);
    if (lane == 0) top_s[t] = top, sum_s[t] = sum, best_s[t] = top > -INFINITY ? best : BCH_NO_TOKEN;
  }
  if (tid < n) token_s[tid] = a.tokens[row0 + tid];
  __syncthreads();
  // The target's probability of token x after token t.
  auto chance = [&](uint32_t t, uint32_t x) {
    if (x >= a.n_vocab || best_s[t] == BCH_NO_TOKEN) return 0.0;
    if (greedy) return x == best_s[t] ? 1.0 : 0.0;
    const float l = logit(a.logits[(uint64_t)(row0 + t) * a.n_vocab + x]);
    return l > -INFINITY ? exp2(((double)l - top_s[t]) * heat64) / sum_s[t] : 0.0;
  };
  if (tid && tid < n) {
    const uint32_t t = parent_of(tid), x = token_s[tid];
    const double p = chance(t, x);
    p_s[tid] = p;
    q_s[tid] = drawn && x < a.n_vocab ? (double)a.draft[(uint64_t)(row0 + t) * a.n_vocab + x] : drawn ? 0.0 : 1.0;
    if (a.chances) a.chances[row0 + tid] = (float)p;
    bool again = false;
    for (uint32_t s = child_of(t); s < tid; s = sibling_of(s)) again |= token_s[s] == x;
    again_s[tid] = again;
  }
  if (tid < n) path_s[tid] = BCH_NO_TOKEN;
  __syncthreads();

  // What is left of p after token t: elements from `from` on, 64 at a time, of the
  // row as weights (times the whole sum where children were drawn, which p - c·q needs
  // normalised; otherwise as they are).  `fallen`: the rejected children.
  uint32_t t = 0, kept = 1;
  double c = 0, left = 1, total = 1;
  auto weight = [&](uint32_t i, float top, float inv) {
    if (i >= a.n_vocab) return 0.f;
    const uint64_t at = (uint64_t)(row0 + t) * a.n_vocab + i;
    const float p = heat.weight(logit(a.logits[at]), top) * inv;
    // (What the target does not have stays at 0, whatever the draft says.)
    return c > 0 && p > 0.f ? fmaxf(fmaf((float)-c, a.draft[at], p), 0.f) : p;
  };
  // The vocabulary in spans of whole 64s, at most kWalkThreads of them; a wave
  // sums every kWalkWaves-th.  Their sums to span_s, the whole's is returned.
  const uint32_t span = (a.n_vocab + kWalkThreads * 64 - 1) / (kWalkThreads * 64) * 64, spans = (a.n_vocab + span - 1) / span;
  auto fallen = [&](uint32_t i) {  // whether element i is a rejected child's token (without a draft)
    for (uint32_t s = child_of(t); s != kKvNone; s = sibling_of(s))
      if (token_s[s] == i) return true;
    return false;
  };
  auto sums = [&](bool without) {
    const float top = fmaxf(top_s[t], -kLargest), inv = (float)(1.0 / sum_s[t]);
    double all = 0;
    for (uint32_t s = wave; s < spans; s += kWalkWaves) {
      double sum = 0;
      for (uint32_t i = s * span + lane; i < (s + 1) * span; i += 64) {
        const float w = weight(i, top, inv);
        sum += without && w > 0.f && fallen(i) ? 0.0 : (double)w;
      }
      sum = wave_sum_f64(sum);
      if (lane == 0) span_s[s] = sum;
      all += sum;
    }
    __syncthreads();
    if (lane == 0) part_s[wave] = all;
    __syncthreads();
    all = 0;
    for (uint32_t w = 0; w < kWalkWaves; w++) all += part_s[w];
    return all;
  };

  if (tid == 0) path_s[0] = 0;
  for (;;) {
    c = 0, left = 1, total = 1;
    uint32_t s = child_of(t);
    for (; s != kKvNone; s = sibling_of(s)) {
      const double u = (double)a.uniforms[row0 + s], p = p_s[s], q = q_s[s];
      if (p > 0 && (greedy ? true : drawn ? u * q * total < (p - c * q) * left : u * total < (again_s[s] ? 0.0 : p))) break;
      if (drawn) {
        if (left > 0) c += total / left;
        if (a.distinct) left -= q;
        total = sums(false);
      } else if (!greedy && !again_s[s]) {
        total -= p;
      }
    }
    if (s == kKvNone) break;
    if (tid == 0) path_s[kept] = s;
    kept++;
    t = s;
  }

  // The next token.
  if (tid == 0) next_s = greedy ? best_s[t] : BCH_NO_TOKEN;
  __syncthreads();
  if (!greedy && best_s[t] != BCH_NO_TOKEN) {
    const bool without = !drawn && child_of(t) != kKvNone;
    total = sums(without);
    bool all = false;  // p itself
    if (!(total > 0)) {
      c = 0;
      all = true;
      total = sums(false);
    }
    // The span in which the sum passes the goal: a thread a span.
    const double goal = (double)a.uniforms[row0] * total;
    double mine = tid < spans ? span_s[tid] : 0, up = mine;
#pragma unroll
    for (int i = 1; i < 64; i *= 2) {
      const double x = __shfl_up(up, i, 64);
      if (lane >= (uint32_t)i) up += x;
    }
    __syncthreads();
    if (lane == 63) part_s[wave] = up;
    __syncthreads();
    double before = 0;
    for (uint32_t w = 0; w < wave; w++) before += part_s[w];
    up += before;
    span_s[tid] = up;  // the sum up to the span's end
    __syncthreads();
    // The first span whose end lies past the goal and that has any weight, or the last
    // that has any.
    uint32_t pick = tid < spans && mine > 0 && up > goal ? tid : ~0u, last = tid < spans && mine > 0 ? tid : 0;
#pragma unroll
    for (int i = 1; i < 64; i *= 2) {
      pick = min(pick, (uint32_t)__shfl_xor((int)pick, i, 64));
      last = max(last, (uint32_t)__shfl_xor((int)last, i, 64));
    }
    __shared__ uint32_t pick_s[kWalkWaves], last_s[kWalkWaves];
    if (lane == 0) pick_s[wave] = pick, last_s[wave] = last;
    __syncthreads();
    if (wave == 0) {
      for (uint32_t w = 0; w < kWalkWaves; w++) pick = min(pick, pick_s[w]), last = max(last, last_s[w]);
      const uint32_t s = pick == ~0u ? last : pick;
      double sum = s ? span_s[s - 1] : 0;
      const float top = fmaxf(top_s[t], -kLargest), inv = (float)(1.0 / sum_s[t]);
      uint32_t found = BCH_NO_TOKEN, some = BCH_NO_TOKEN;
      for (uint32_t i0 = s * span; i0 < (s + 1) * span && found == BCH_NO_TOKEN; i0 += 64) {
        const uint32_t i = i0 + lane;
        const float w = weight(i, top, inv);
        const double x = without && !all && w > 0.f && fallen(i) ? 0.0 : (double)w;
        double run = x;
#pragma unroll
        for (int k = 1; k < 64; k *= 2) {
          const double y = __shfl_up(run, k, 64);
          if (lane >= (uint32_t)k) run += y;
        }
        const uint64_t past = __builtin_amdgcn_ballot_w64(x > 0 && sum + run > goal), any = __builtin_amdgcn_ballot_w64(x > 0);
        if (past) found = i0 + __ffsll((unsigned long long)past) - 1;
        if (any) some = i0 + 63 - __clzll((long long)any);
        sum += __shfl(run, 63, 64);
      }
      if (lane == 0) next_s = found != BCH_NO_TOKEN ? found : some;
    }
    __syncthreads();
  }
  if (tid < n) a.path[row0 + tid] = path_s[tid];
  if (tid == 0) {
    a.kept[blockIdx.x] = kept;
    a.next[blockIdx.x] = next_s;
    if (a.chances) a.chances[row0] = next_s == BCH_NO_TOKEN ? 0.f : (float)chance(t, next_s);
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
  a.n_pieces = div_ceil(n_vocab, kRowPiece);
  a.distinct = drafts->distinct != 0;
  if ((uint64_t)a.n_rows * a.n_pieces >= 1u << 23) return fail(BCH_ERR_ARGUMENT, "verify_drafts: too many logits");
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
  void *scratch;
  BCH_TRY(ctx_scratch(ctx, std::max<uint64_t>(rows * a.n_pieces * sizeof(VerifyPiece), 16), &scratch));
  a.pieces = static_cast<VerifyPiece *>(scratch);
  return launch(ctx, {"verify_drafts", a.n_rows, n_vocab, 0}, [&](hipStream_t st) {
    if (!n_seqs) return;
    kv_plan_use(ctx, plan);
    a.seqs = plan->d_seqs + first;
    a.nodes = plan->d_nodes ? plan->d_nodes + a.row0 : nullptr;
    if (a.n_rows) k_verify_rows<<<a.n_rows * a.n_pieces, kRowThreads, 0, st>>>(a);
    k_verify_walk<<<n_seqs, kWalkThreads, 0, st>>>(a);
  });
}
