// Rotary positions of a batch's queries and keys, each token's from its plan,
// after an RMS norm of the head where one is wanted.
//
// Pair j of a head at position t turns by t·f_j radians.  An f32 product is off
// by up to t·2^-25 radians, so the angle is taken in turns instead: F_j = f_j / 2π
// is kept in 2^-64 of a turn, and t·F_j mod 2^64 is exactly what is left of it
// after all whole turns.  The nearest quarter turn is split off as two bits, the
// rest (an eighth of a turn either way) is exact to 2^-32 of a turn as an
// integer and to 2^-24 of itself as a float, and its sine and cosine are their series to
// x^9 and x^10, whose next terms are below 2^-28.
//
// Bound by the bytes: 7,362 tokens, 40 heads of 128, 301 MB, 61.5 us (4.9 TB/s, a copy's
// rate); few tokens by latency, one of 40 heads of 64 2.9 us, 437 of 10 heads of 256 5.0.
#include <algorithm>
#include <cmath>
#include <memory>
#include <new>

#include "device.h"
#include "kernels.h"
#include "kv_cache.h"
#include "runtime.h"

struct bch_rope {
  bch_ctx *ctx;
  uint32_t layout, n_rot;
  float magnitude;
  uint64_t *turns;  // [n_rot / 2] on the device
};

namespace bch {

constexpr uint32_t kRopeThreads = 256, kRopeMaxRot = 256, kRopeMaxHeads = 1u << 16;

// cos and sin of t / 2^64 turns.
__device__ __forceinline__ float2 cos_sin(uint64_t t) {
  const uint32_t h = (uint32_t)(t >> 32), quarter = (h + 0x20000000u) >> 30;
  const float x = (float)(int32_t)(h - (quarter << 30)) * (float)(6.283185307179586476925 * 0x1p-32), y = x * x;
  float s = fmaf(y, 1.f / 362880, -1.f / 5040), c = fmaf(y, -1.f / 3628800, 1.f / 40320);
  s = fmaf(s, y, 1.f / 120), c = fmaf(c, y, -1.f / 720);
  s = fmaf(s, y, -1.f / 6), c = fmaf(c, y, 1.f / 24);
  s = fmaf(s * y, x, x), c = fmaf(c, y, -0.5f);
  c = fmaf(c, y, 1.f);
  const float a = quarter & 1 ? s : c, b = quarter & 1 ? c : s;
  return {(quarter + 1) & 2 ? -a : a, quarter & 2 ? -b : b};
}

// Four floats, with STREAM past the caches.
template <bool STREAM>
__device__ __forceinline__ void put4(float *p, const float *z) {
  typedef float f4 __attribute__((ext_vector_type(4)));
  const f4 v = {z[0], z[1], z[2], z[3]};
  if constexpr (STREAM)
    __builtin_nontemporal_store(v, reinterpret_cast<f4 *>(p));
  else
    *reinterpret_cast<f4 *>(p) = v;
}

struct RopeSide {
  const float *from;
  float *to;
  const float *norm;  // or null
  uint32_t n_heads, head_stride, from_stride, to_stride;
  float eps;
};
struct RopeArgs {
  const KvStoreItem *items;
  const KvNode *nodes;  // null: tokens of an item are at consecutive positions
  const uint64_t *turns;
  RopeSide side[2];  // queries and keys
  uint32_t half;     // pairs
  float magnitude;
};

// A workgroup takes rows (a head of a token) of one block's tokens, HD / 8 lanes
// each, head after head: where the tokens divide the rows of a round, every
// round's row of a lane has the same token, whose angles the lane keeps.  QUADS: a
// lane has two pieces of four elements, and pairs 4·lane .. + 3 where those turn;
// else up to 8 pairs and single elements, one by one, for any n_rot.
template <uint32_t HD, uint32_t LAYOUT, bool QUADS, bool STREAM>
__global__ __launch_bounds__(kRopeThreads) void k_rope(RopeArgs a) {
  constexpr uint32_t LANES = HD / 8, ROWS = kRopeThreads / LANES;
  const KvStoreItem it = a.items[blockIdx.x];
  const uint32_t lane = threadIdx.x % LANES, n = it.n, magic = n > 1 ? 0xffffffffu / n + 1 : 0;
  const uint32_t rows = n * (a.side[0].n_heads + a.side[1].n_heads), n_rot = 2 * a.half;
  // Element of the first of a unit's pair and the distance to the second.
  auto place = [&](uint32_t u) { return LAYOUT == BCH_ROPE_PAIRS ? 2 * u : u; };
  const uint32_t apart = LAYOUT == BCH_ROPE_PAIRS ? 1 : a.half;
  float co[QUADS ? 4 : 8], si[QUADS ? 4 : 8];
  uint32_t known = ~0u;
  for (uint32_t r = blockIdx.y * ROWS + threadIdx.x / LANES; r < rows; r += gridDim.y * ROWS) {
    uint32_t head = n > 1 ? __umulhi(r, magic) : r;
    const uint32_t token = r - head * n;
    const bool key = head >= a.side[0].n_heads;
    const RopeSide &s = a.side[key];
    head -= key ? a.side[0].n_heads : 0;
    const float *from = s.from + (uint64_t)(it.row + token) * s.from_stride + (uint64_t)head * s.head_stride;
    float *to = s.to + (uint64_t)(it.row + token) * s.to_stride + (uint64_t)head * HD;
    // The lane's elements: x[i] and x[i + 4] (QUADS and halves), x[2i] and x[2i + 1] (QUADS and pairs) or
    // x[i] and y[i] are pairs.
    float x[8], y[8];
    uint32_t q0 = 0, q1 = 0;
    if constexpr (QUADS) {
      if (LAYOUT == BCH_ROPE_PAIRS)
        q0 = 8 * lane, q1 = q0 + 4;
      else if (4 * lane < a.half)
        q0 = 4 * lane, q1 = a.half + 4 * lane;
      else
        q0 = 8 * lane, q1 = q0 + 4;
      const float4 f = *reinterpret_cast<const float4 *>(from + q0), g = *reinterpret_cast<const float4 *>(from + q1);
      x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w, x[4] = g.x, x[5] = g.y, x[6] = g.z, x[7] = g.w;
    } else {
#pragma unroll
      for (uint32_t i = 0; i < 8; i++) {
        const uint32_t u = lane + LANES * i, single = n_rot + (u - a.half);
        x[i] = u < a.half ? from[place(u)] : single < HD ? from[single] : 0.f;
        y[i] = u < a.half ? from[place(u) + apart] : 0.f;
      }
    }
    if (token != known) {
      known = token;
      const uint64_t t = a.nodes ? a.nodes[it.row + token].position : it.pos + token;
#pragma unroll
      for (uint32_t i = 0; i < (QUADS ? 4 : 8); i++) {
        const uint32_t j = QUADS ? 4 * lane + i : lane + LANES * i;
        const float2 v = cos_sin(t * a.turns[min(j, a.half - 1)]);
        co[i] = j < a.half ? v.x * a.magnitude : 1.f;
        si[i] = j < a.half ? v.y * a.magnitude : 0.f;
      }
    }
    if (s.norm) {
      float sum = 0.f;
#pragma unroll
      for (uint32_t i = 0; i < 8; i++) {
        sum = fmaf(x[i], x[i], sum);
        if constexpr (!QUADS) sum = fmaf(y[i], y[i], sum);
      }
      const float scale = rsqrtf(group_sum<(int)LANES>(sum) * (1.f / HD) + s.eps);
      if constexpr (QUADS) {
        const float4 f = *reinterpret_cast<const float4 *>(s.norm + q0), g = *reinterpret_cast<const float4 *>(s.norm + q1);
        const float w[8] = {f.x, f.y, f.z, f.w, g.x, g.y, g.z, g.w};
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) x[i] *= scale * w[i];
      } else {
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) {
          const uint32_t u = lane + LANES * i, single = n_rot + (u - a.half);
          if (u < a.half)
            x[i] *= scale * s.norm[place(u)], y[i] *= scale * s.norm[place(u) + apart];
          else if (single < HD)
            x[i] *= scale * s.norm[single];
        }
      }
    }
    if constexpr (QUADS) {
      float z[8];
#pragma unroll
      for (uint32_t i = 0; i < 4; i++) {
        const uint32_t p = LAYOUT == BCH_ROPE_PAIRS ? 2 * i : i, q = LAYOUT == BCH_ROPE_PAIRS ? p + 1 : i + 4;
        // (Elements that do not turn stay as they are, whatever they hold.)
        const bool turns = 4 * lane + i < a.half;
        z[p] = turns ? fmaf(x[p], co[i], -x[q] * si[i]) : x[p];
        z[q] = turns ? fmaf(x[p], si[i], x[q] * co[i]) : x[q];
      }
      put4<STREAM>(to + q0, z);
      put4<STREAM>(to + q1, z + 4);
    } else {
#pragma unroll
      for (uint32_t i = 0; i < 8; i++) {
        const uint32_t u = lane + LANES * i, single = n_rot + (u - a.half);
        if (u < a.half) {
          to[place(u)] = fmaf(x[i], co[i], -y[i] * si[i]);
          to[place(u) + apart] = fmaf(x[i], si[i], y[i] * co[i]);
        } else if (single < HD) {
          to[single] = x[i];
        }
      }
    }
  }
}

static int check_spec(const bch_rope_spec *s) {
  if (!s) return fail(BCH_ERR_ARGUMENT, "rope: no spec");
  if (s->layout > BCH_ROPE_PAIRS || s->scaling > BCH_ROPE_BY_PARTS)
    return fail(BCH_ERR_ARGUMENT, "rope: layout %u, scaling %u", s->layout, s->scaling);
  if (!s->n_rot || s->n_rot % 2 || s->n_rot > kRopeMaxRot)
    return fail(BCH_ERR_ARGUMENT, "rope: %u elements turn: an even number from 2 to %u is wanted", s->n_rot, kRopeMaxRot);
  auto above_0 = [](double x) { return x > 0 && std::isfinite(x); };
  if (!above_0(s->theta)) return fail(BCH_ERR_ARGUMENT, "rope: theta %g", s->theta);
  if (s->scaling != BCH_ROPE_PLAIN && !above_0(s->factor)) return fail(BCH_ERR_ARGUMENT, "rope: factor %g", s->factor);
  if (s->scaling == BCH_ROPE_BY_PARTS &&
      (!s->n_original || !std::isfinite(s->slow) || !std::isfinite(s->fast) || s->slow >= s->fast))
    return fail(BCH_ERR_ARGUMENT, "rope: %u positions, from %g to %g turns", s->n_original, s->slow, s->fast);
  if (!std::isfinite(s->magnitude) || std::fabs(s->magnitude) > 1e30)
    return fail(BCH_ERR_ARGUMENT, "rope: magnitude %g", s->magnitude);
  return BCH_OK;
}

static double frequency(const bch_rope_spec &s, uint32_t j) {
  const double f = std::pow(s.theta, -2.0 * j / s.n_rot);
  if (s.scaling == BCH_ROPE_LINEAR) return f / s.factor;
  if (s.scaling != BCH_ROPE_BY_PARTS) return f;
  const double turns = s.n_original * f / 6.283185307179586476925;
  const double w = std::min(std::max((turns - s.slow) / (s.fast - s.slow), 0.0), 1.0);
  return f * (w + (1 - w) / s.factor);
}

// Radians a position as 2^-64 of a turn, whole turns left out.
static uint64_t turns_of(double radians) {
  const long double turns = radians / 6.283185307179586476925286766559L;
  const long double part = (turns - std::floor(turns)) * 0x1p64L;
  return part >= 0x1p64L ? 0 : (uint64_t)part;
}

}  // namespace bch

using namespace bch;

extern "C" int bch_rope_frequencies(const bch_rope_spec *spec, double *out) {
  BCH_TRY(check_spec(spec));
  if (!out) return fail(BCH_ERR_ARGUMENT, "rope: nowhere to store the frequencies");
  for (uint32_t j = 0; j < spec->n_rot / 2; j++) out[j] = frequency(*spec, j);
  return BCH_OK;
}

extern "C" int bch_rope_new(bch_ctx *ctx, const bch_rope_spec *spec, const double *frequencies, bch_rope **out) {
  if (!out) return fail(BCH_ERR_ARGUMENT, "rope: nowhere to store it");
  *out = nullptr;
  BCH_TRY(check_spec(spec));
  uint64_t turns[kRopeMaxRot / 2];
  for (uint32_t j = 0; j < spec->n_rot / 2; j++) {
    const double f = frequencies ? frequencies[j] : frequency(*spec, j);
    if (!std::isfinite(f)) return fail(BCH_ERR_ARGUMENT, "rope: frequency %u is %g", j, f);
    turns[j] = turns_of(f);
  }
  if (!ctx) return fail(BCH_ERR_ARGUMENT, "rope: no backend");
  std::unique_ptr<bch_rope> rope(new (std::nothrow) bch_rope{ctx, spec->layout, spec->n_rot, (float)spec->magnitude, nullptr});
  if (!rope) return fail(BCH_ERR_ALLOCATION, "rope: out of host memory");
  void *p = nullptr;
  if (hipMalloc(&p, spec->n_rot / 2 * 8) != hipSuccess) {
    (void)hipGetLastError();
    return fail(BCH_ERR_ALLOCATION, "rope: cannot allocate its frequencies");
  }
  // Done before this returns, so before any launch that reads it.
  if (hipMemcpy(p, turns, spec->n_rot / 2 * 8, hipMemcpyHostToDevice) != hipSuccess ||
      hipStreamSynchronize(nullptr) != hipSuccess) {
    hipFree(p);
    return fail(BCH_ERR_EXECUTION, "rope: host-to-device copy failed");
  }
  rope->turns = static_cast<uint64_t *>(p);
  *out = rope.release();
  return BCH_OK;
}

extern "C" void bch_rope_free(bch_rope *rope) {
  if (!rope) return;
  hipStreamSynchronize(rope->ctx->stream);
  hipFree(rope->turns);
  delete rope;
}

// One side's rows, and where they lie.
struct Span {
  const float *at;
  uint64_t bytes;
  uint32_t width, stride;
};

static int rope_side(bch_ctx *ctx, const bch_kv_plan *plan, const bch_rope_rows *r, RopeSide *side, Span *from, Span *to) {
  const uint32_t hd = plan->shape.head_dim;
  if (!r->n_heads || r->n_heads > kRopeMaxHeads) return fail(BCH_ERR_ARGUMENT, "rope_paged: %u heads", r->n_heads);
  if (r->head_stride < hd || r->head_stride % 4 || r->head_stride > 1u << 14)
    return fail(BCH_ERR_ARGUMENT, "rope_paged: heads of %u floats %u apart", hd, r->head_stride);
  const uint32_t width = (r->n_heads - 1) * r->head_stride + hd;
  float *p;
  BCH_TRY(kv_plan_rows(ctx, "rope_paged", plan, r->from, width, r->from_stride, &p));
  BCH_TRY(kv_plan_rows(ctx, "rope_paged", plan, r->to, r->n_heads * hd, r->to_stride, &side->to));
  side->from = p;
  if (r->norm.buffer) {
    BCH_TRY(view_ptr(ctx, "rope_paged", r->norm, hd * 4, &side->norm));
    if (reinterpret_cast<uintptr_t>(side->norm) % 16) return fail(BCH_ERR_ARGUMENT, "rope_paged: the norm must be 16-byte aligned");
  }
  side->n_heads = r->n_heads;
  side->head_stride = r->head_stride;
  side->from_stride = r->from_stride;
  side->to_stride = r->to_stride;
  side->eps = r->eps;
  *from = {side->from, kv_rows_bytes(plan, width, r->from_stride), width, r->from_stride};
  *to = {side->to, kv_rows_bytes(plan, r->n_heads * hd, r->to_stride), r->n_heads * hd, r->to_stride};
  return BCH_OK;
}

// Whether no float of the one's rows is one of the other's.
static bool rope_apart(const Span &a, const Span &b) {
  if (!kv_overlap(a.at, a.bytes, b.at, b.bytes)) return true;
  if (a.stride != b.stride) return false;
  // Side by side in rows of one stride.
  const uint64_t d = a.at < b.at ? (uint64_t)(b.at - a.at) % a.stride : (a.stride - (uint64_t)(a.at - b.at) % a.stride) % a.stride;
  return d >= a.width && d <= a.stride - b.width;
}

extern "C" int bch_rope_paged(bch_ctx *ctx, const bch_rope *rope, const bch_kv_plan *plan, const bch_rope_rows *q,
                              const bch_rope_rows *k) {
  if (!rope) return fail(BCH_ERR_ARGUMENT, "rope_paged: no rope");
  if (rope->ctx != ctx) return fail(BCH_ERR_FOREIGN_BUFFER, "rope_paged: the rope belongs to another backend");
  BCH_TRY(kv_plan_ready(ctx, "rope_paged", plan));
  const uint32_t hd = plan->shape.head_dim;
  if (rope->n_rot > hd) return fail(BCH_ERR_ARGUMENT, "rope_paged: %u elements of heads of %u turn", rope->n_rot, hd);
  RopeArgs a{};
  Span from[2] = {}, to[2] = {};
  const bch_rope_rows *const rows[2] = {q, k};
  for (int i = 0; i < 2; i++)
    if (rows[i]) BCH_TRY(rope_side(ctx, plan, rows[i], &a.side[i], &from[i], &to[i]));
  for (int i = 0; i < 2; i++)
    for (int j = 0; j < 2; j++) {
      if (!rows[i] || !rows[j]) continue;
      const bool in_place = i == j && to[i].at == from[i].at && to[i].stride == from[i].stride && to[i].width == from[i].width;
      if (!in_place && !rope_apart(to[i], from[j]))
        return fail(BCH_ERR_ARGUMENT, "rope_paged: rows that are written lie over rows that are read");
      if (i < j && !rope_apart(to[i], to[j]))
        return fail(BCH_ERR_ARGUMENT, "rope_paged: the queries and the keys are written to one place");
      if (a.side[j].norm && kv_overlap(to[i].at, to[i].bytes, a.side[j].norm, hd * 4))
        return fail(BCH_ERR_ARGUMENT, "rope_paged: rows that are written lie over a norm");
    }
  const uint32_t heads = a.side[0].n_heads + a.side[1].n_heads;
  return launch(ctx, {"rope_paged", plan->n_tokens, heads * hd, 0}, [&](hipStream_t st) {
    if (!plan->n_store || !heads) return;
    kv_plan_use(ctx, plan);
    a.items = plan->d_store;
    a.nodes = plan->d_nodes;
    a.turns = rope->turns;
    a.half = rope->n_rot / 2;
    a.magnitude = rope->magnitude;
    // Rows that no L2 holds until they are read go past the caches (151 MB of them: 62 us instead of
    // 71; 4.5 MB are read back from the L2 and take 5 us either way).
    const bool stream = (uint64_t)plan->n_tokens * heads * hd * 4 > 32u << 20;
    const bool quads = rope->n_rot % (rope->layout == BCH_ROPE_PAIRS ? 4 : 8) == 0;
    auto go = [&](auto width, auto layout, auto by_quads, auto streams) {
      constexpr uint32_t HD = decltype(width)::value, ROWS = kRopeThreads / (HD / 8);
      const uint32_t most = div_ceil(heads * std::min(kKvBlock, plan->n_tokens), ROWS);
      const dim3 grid(plan->n_store, std::max(1u, std::min(most, div_ceil(8 * 256, plan->n_store))));
      k_rope<HD, decltype(layout)::value, decltype(by_quads)::value, decltype(streams)::value><<<grid, kRopeThreads, 0, st>>>(a);
    };
    auto with_layout = [&](auto width) {
      auto with_quads = [&](auto layout) {
        if (quads && stream)
          go(width, layout, std::true_type{}, std::true_type{});
        else if (quads)
          go(width, layout, std::true_type{}, std::false_type{});
        else
          go(width, layout, std::false_type{}, std::false_type{});
      };
      if (rope->layout == BCH_ROPE_PAIRS)
        with_quads(std::integral_constant<uint32_t, BCH_ROPE_PAIRS>{});
      else
        with_quads(std::integral_constant<uint32_t, BCH_ROPE_HALVES>{});
    };
    if (hd == 64)
      with_layout(std::integral_constant<uint32_t, 64>{});
    else if (hd == 128)
      with_layout(std::integral_constant<uint32_t, 128>{});
    else
      with_layout(std::integral_constant<uint32_t, 256>{});
  });
}
