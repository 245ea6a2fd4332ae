// The rules of a batch's rows on their logits, before the sampler: penalties
// for the tokens of the row's history, biases, and a grammar's mask.
//
// With c the times that a token occurs in the history,
//   y = (x > 0 ? x / repeat : x·repeat) − (presence + frequency·c)  for c > 0, else x,
// then y + b for every bias (token, b) of the row in list order, then −inf
// where the mask's bit is 0.
//
// One launch and one pass: a workgroup owns a slice of one row's vocabulary,
// counts the whole history's tokens that fall into it in LDS (integers: the
// order of the atomics changes nothing), and reads and writes its logits once.
// That a row's history is read by each of its slices costs less than counters
// in memory would: 4 bytes a token out of the L2 against 8 bytes a logit.
// Bound by the logits' bytes: 96 rows of 151,936 with histories of 2,000 tokens
// take 30 us (4.0 TB/s); a single row by latency (5.9 us).
#include <cmath>

#include "device.h"
#include "kernels.h"
#include "runtime.h"

namespace bch {

constexpr uint32_t kEditPer = 8;  // logits of a thread

struct EditArgs {
  const float *logits;
  float *out;
  const bch_logit_row *rows;
  const uint32_t *history, *bias_tokens, *masks;
  const float *bias_values;
  uint32_t n_vocab, n_history, n_bias, n_masks, slices;
};

// Slices of THREADS·PER tokens.
template <uint32_t THREADS>
__global__ __launch_bounds__(THREADS) void k_logits_edit(EditArgs a) {
  constexpr uint32_t PER = kEditPer, SLICE = THREADS * PER;
  __shared__ uint32_t count_s[SLICE];  // then the logits as the biases change them
  __shared__ uint32_t owner_s[SLICE];
  const uint32_t row = blockIdx.x / a.slices, base = blockIdx.x % a.slices * SLICE, tid = threadIdx.x;
  const uint32_t len = min(SLICE, a.n_vocab - base);
  const bch_logit_row r = a.rows[row];
  const uint64_t at = (uint64_t)row * a.n_vocab + base;
  // (Streamed past the caches: 30 us instead of 36 for 96 rows of 151,936 with
  // histories of 2,000 tokens.)
  float x[PER];
#pragma unroll
  for (uint32_t j = 0; j < PER; j++) {
    const uint32_t i = tid + THREADS * j;
    x[j] = i < len ? __builtin_nontemporal_load(a.logits + at + i) : 0.f;
  }
  // Lists never leave the buffers, whatever the row says.
  const uint32_t h0 = min(r.history_at, a.n_history), hn = min(r.history_len, a.n_history - h0);
  const uint32_t b0 = min(r.bias_at, a.n_bias), bn = min(r.bias_len, a.n_bias - b0);
  if (hn) {
    for (uint32_t i = tid; i < SLICE; i += THREADS) count_s[i] = 0;
    __syncthreads();
    const uint32_t *history = a.history + h0;
    constexpr uint32_t N = 4;  // tokens in flight
    for (uint32_t i = tid; i < hn; i += THREADS * N) {
      uint32_t t[N];
#pragma unroll
      for (uint32_t j = 0; j < N; j++) t[j] = i + THREADS * j < hn ? history[i + THREADS * j] - base : ~0u;
#pragma unroll
      for (uint32_t j = 0; j < N; j++)
        if (t[j] < len) atomicAdd(&count_s[t[j]], 1u);  // (a token below base has wrapped past the slice)
    }
    __syncthreads();
#pragma unroll
    for (uint32_t j = 0; j < PER; j++) {
      const uint32_t c = count_s[tid + THREADS * j];
      if (c) x[j] = (x[j] > 0.f ? x[j] / r.repeat : x[j] * r.repeat) - (r.presence + r.frequency * (float)c);
    }
  }
  if (bn) {
    float *y_s = reinterpret_cast<float *>(count_s);
#pragma unroll
    for (uint32_t j = 0; j < PER; j++) {
      y_s[tid + THREADS * j] = x[j];  // (each thread's own counters)
      owner_s[tid + THREADS * j] = ~0u;
    }
    __syncthreads();
    // THREADS biases at a time, each in turn added by the lowest thread that has
    // one for its token: one round, or as many as a token is named.
    for (uint32_t i0 = 0; i0 < bn; i0 += THREADS) {
      const uint32_t i = i0 + tid;
      const uint32_t t = i < bn ? a.bias_tokens[b0 + i] - base : ~0u;
      bool waiting = t < len;
      while (__syncthreads_or(waiting)) {
        if (waiting) atomicMin(&owner_s[t], tid);
        __syncthreads();
        const bool mine = waiting && owner_s[t] == tid;
        __syncthreads();
        if (mine) {
          y_s[t] += a.bias_values[b0 + i];
          owner_s[t] = ~0u;
          waiting = false;
        }
      }
    }
#pragma unroll
    for (uint32_t j = 0; j < PER; j++) x[j] = y_s[tid + THREADS * j];
  }
  const bool masked = r.mask != BCH_NO_MASK, known = r.mask < a.n_masks;
  const uint32_t *mask = known ? a.masks + (uint64_t)r.mask * ((a.n_vocab + 31) / 32) : nullptr;
#pragma unroll
  for (uint32_t j = 0; j < PER; j++) {
    const uint32_t i = tid + THREADS * j;
    if (i >= len) continue;
    const uint32_t t = base + i;
    const bool allowed = !masked || (known && (mask[t / 32] >> (t % 32) & 1));
    __builtin_nontemporal_store(allowed ? x[j] : -INFINITY, a.out + at + i);
  }
}

}  // namespace bch

using namespace bch;

extern "C" int bch_logits_edit(bch_ctx *ctx, bch_view logits, bch_view out, uint32_t n_rows, uint32_t n_vocab,
                               const bch_logit_rules *rules) {
  if (!rules) return fail(BCH_ERR_ARGUMENT, "logits_edit: no rules");
  if (!n_vocab || n_vocab > 1u << 30) return fail(BCH_ERR_ARGUMENT, "logits_edit: rows of %u logits", n_vocab);
  // (The kernel's places in a list and a step behind them are 32 bits.)
  if (rules->n_history > 1u << 30 || rules->n_bias > 1u << 30)
    return fail(BCH_ERR_ARGUMENT, "logits_edit: lists of more than 2^30 entries");
  // Slices of 4,096 logits for long histories, of which each slice reads all, and
  // of 2,048 for short ones, whose rows make more workgroups: 96 rows of 151,936
  // with 2,000 tokens on average 29 us and 32, with 1 token 22 and 22; one row of
  // 65,536 with 600 tokens 6.4 and 5.8.  (The same inputs each time; 16 logits a
  // thread instead of eight: 39 and 42 instead of 29 and 32.)
  const bool long_history = n_rows && rules->n_history / n_rows > 1024;
  const uint32_t threads = long_history ? 512 : 256, slices = div_ceil(n_vocab, threads * kEditPer);
  if ((uint64_t)n_rows * slices >= 1u << 23) return fail(BCH_ERR_ARGUMENT, "logits_edit: too many logits");
  EditArgs a{};
  a.n_vocab = n_vocab;
  a.n_history = rules->n_history;
  a.n_bias = rules->n_bias;
  a.n_masks = rules->n_masks;
  a.slices = slices;
  const uint64_t bytes = (uint64_t)n_rows * n_vocab * 4;
  BCH_TRY(view_ptr(ctx, "logits_edit", logits, bytes, &a.logits));
  BCH_TRY(view_ptr(ctx, "logits_edit", out, bytes, &a.out));
  BCH_TRY(view_ptr(ctx, "logits_edit", rules->rows, (uint64_t)n_rows * sizeof(bch_logit_row), &a.rows));
  if (rules->n_history) BCH_TRY(view_ptr(ctx, "logits_edit", rules->history, (uint64_t)rules->n_history * 4, &a.history));
  if (rules->n_bias) {
    BCH_TRY(view_ptr(ctx, "logits_edit", rules->bias_tokens, (uint64_t)rules->n_bias * 4, &a.bias_tokens));
    BCH_TRY(view_ptr(ctx, "logits_edit", rules->bias_values, (uint64_t)rules->n_bias * 4, &a.bias_values));
  }
  if (rules->n_masks)
    BCH_TRY(view_ptr(ctx, "logits_edit", rules->masks, (uint64_t)rules->n_masks * ((n_vocab + 31) / 32) * 4, &a.masks));
  for (const void *p : {(const void *)a.logits, (const void *)a.out, (const void *)a.rows, (const void *)a.history,
                        (const void *)a.bias_tokens, (const void *)a.bias_values, (const void *)a.masks})
    if (reinterpret_cast<uintptr_t>(p) % 4) return fail(BCH_ERR_ARGUMENT, "logits_edit: operands must be 4-byte aligned");
  const uintptr_t from = reinterpret_cast<uintptr_t>(a.logits), to = reinterpret_cast<uintptr_t>(a.out);
  auto over = [&](const void *list, uint64_t list_bytes) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(list);
    return x < to + bytes && to < x + list_bytes;
  };
  if (from != to && over(a.logits, bytes))
    return fail(BCH_ERR_ARGUMENT, "logits_edit: the outputs lie over the logits (the same place or another is wanted)");
  // (Slices read the lists while others write.)
  if (over(a.rows, (uint64_t)n_rows * sizeof(bch_logit_row)) || over(a.history, (uint64_t)a.n_history * 4) ||
      over(a.bias_tokens, (uint64_t)a.n_bias * 4) || over(a.bias_values, (uint64_t)a.n_bias * 4) ||
      over(a.masks, (uint64_t)a.n_masks * ((n_vocab + 31) / 32) * 4))
    return fail(BCH_ERR_ARGUMENT, "logits_edit: the outputs lie over the rules");
  return launch(ctx, {"logits_edit", n_rows, n_vocab, 0}, [&](hipStream_t s) {
    if (!n_rows) return;
    if (long_history)
      k_logits_edit<512><<<n_rows * a.slices, 512, 0, s>>>(a);
    else
      k_logits_edit<256><<<n_rows * a.slices, 256, 0, s>>>(a);
  });
}
