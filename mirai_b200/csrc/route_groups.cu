// Group-limited routing: top-k experts inside the best groups of experts, and
// the gradient of the routing weights with respect to the logits.
//
//   s = sigmoid(l) or softmax(l);  key = s + bias, or l itself without a bias
//   group score = the largest key of a group, or the sum of its two largest s + bias
//   the top_groups best groups stay; in them the k largest keys (ties: lowest id)
//   w_j = route_scale * s_j / den   (the renormalisations of route_topk)
//
// Decisions are those of 64-bit arithmetic: a row is decided in fp32 together
// with a bound on the fp32 error, and a row where two compared values lie within
// it is decided again in 64 bits.  How many do depends on the inputs: 0.2 % of rows of sigmoid
// scores of logits of deviation 1.2 with a bias; of softmax scores, whose bound follows the row's largest,
// 15 % where logits of deviation 4 meet biases of 1e-4 ([65536, 128]: 64 us for 47).  Without a bias,
// experts and group maxima are ranked by the logits themselves, which is exact.
//
// W lanes hold a token's experts, so a warp routes 32 / W tokens: each group on
// whole lanes (a power of two of them), PER experts per lane, so that expert
// order is lane order, group scores are butterflies inside a group, and ties
// resolve to the lowest lane.
//
// route_fast (up to 32 experts per lane) ranks 32-bit words of the key's leading bits
// and the expert's id: a lane sorts its words by a network of integer minima and
// maxima, and k + 1 rounds take the largest head.  What it cannot decide, the whole
// warp decides one row after the other in 64 bits (route_exact), and every row with more experts per
// lane (from 561 experts on, in a number of groups that is no power of two).
#include "common.cuh"

namespace mirai {
namespace rg {

constexpr int kMaxTopK = 16;
constexpr int kMaxGroups = 32;
constexpr int kMaxExperts = 1024;

struct Args {
  const void* logits;
  const float* bias;
  int64_t T;
  int E, k, G, top_groups;
  int gs;       // experts per group
  int shift;    // log2 of the lanes per group
  int per;      // experts per lane, <= PER
  int shift32, per32;  // the same with a whole warp per token
  int score;    // MIRAI_SCORE_*
  int vec;      // rows can be read 16 bytes at a time
  int vec_bias;
  int id_bits;  // bits of an expert id
  int top2;     // group score: 1 the two best scores, 0 the best key
  int norm;     // MIRAI_NORM_*
  float scale;
  int64_t* idx;
  float* w;
};

__device__ __forceinline__ float load_logit(const float* p) { return __ldg(p); }
__device__ __forceinline__ float load_logit(const __nv_bfloat16* p) { return __bfloat162float(*p); }

// Order-preserving integers (larger is better, 0 below every value): -0 counts as 0.
__device__ __forceinline__ uint32_t order(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t order(double x) {
  const uint64_t b = (uint64_t)__double_as_longlong(x + 0.0);
  return b >> 63 ? ~b : b | (1ull << 63);
}

template <int W, typename V> __device__ __forceinline__ V max_lanes(V v) {
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) {
    v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  }
  return v;
}
template <int W, typename V> __device__ __forceinline__ V sum_lanes(V v) {
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The weights of the selected scores: what they are divided by and multiplied by
// (the formulas of route_topk), and whether the divisor follows their sum.
template <typename F> __device__ __forceinline__ void denominator(int norm, int k, float route_scale, F sum, F& den,
                                                                  F& scale, bool& follows) {
  den = F(1);
  scale = F(route_scale);
  follows = false;
  if (norm == MIRAI_NORM_CLAMP) {
    follows = sum >= F(1e-20f);
    den = follows ? sum : F(1e-20f);
    scale = F(1);
  } else if (norm == MIRAI_NORM_EPS) {
    if (k > 1) {
      follows = true;
      den = sum + F(1e-20f);
    }
  } else if (norm == MIRAI_NORM_L1) {
    follows = sum >= F(1e-12f);
    den = follows ? sum : F(1e-12f);
  }
  if (sum != sum) den = sum;  // NaN scores stay NaN
}

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
constexpr float kLog2e = 1.4426950408889634f;

// PER consecutive values of a row, -inf past the first n of them.  Whole rows of vectors
// (vec) are read 16 bytes at a time.
template <int PER> __device__ __forceinline__ void load_row(const float* p, int n, bool vec, float (&v)[PER]) {
  if (vec) {
#pragma unroll
    for (int i = 0; i < PER; i += 4) {
      float4 x = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      if (i < n) x = __ldg(reinterpret_cast<const float4*>(p + i));
      v[i] = x.x, v[i + 1] = x.y, v[i + 2] = x.z, v[i + 3] = x.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) v[i] = i < n ? __ldg(p + i) : -INFINITY;
  }
}
template <int PER> __device__ __forceinline__ void load_row(const __nv_bfloat16* p, int n, bool vec, float (&v)[PER]) {
  if (vec) {
#pragma unroll
    for (int i = 0; i < PER; i += 4) {
      uint2 x = make_uint2(0xff80ff80u, 0xff80ff80u);
      if (i < n) x = __ldg(reinterpret_cast<const uint2*>(p + i));
      v[i] = bf16_lo(x.x), v[i + 1] = bf16_hi(x.x), v[i + 2] = bf16_lo(x.y), v[i + 3] = bf16_hi(x.y);
    }
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) v[i] = i < n ? __bfloat162float(p[i]) : -INFINITY;
  }
}

// Descending order by compare-exchanges that no data decides: Batcher's odd-even
// merge sort (19 exchanges of 8 words, 63 of 16).
template <int N> __device__ __forceinline__ void sort_desc(uint32_t (&v)[N]) {
#pragma unroll
  for (int p = 1; p < N; p *= 2) {
#pragma unroll
    for (int q = p; q > 0; q /= 2) {
#pragma unroll
      for (int j = q % p; j + q < N; j += 2 * q) {
#pragma unroll
        for (int i = 0; i < q; ++i) {
          if (i + j + q < N && (i + j) / (2 * p) == (i + j + q) / (2 * p)) {
            const uint32_t hi = max(v[i + j], v[i + j + q]), lo = min(v[i + j], v[i + j + q]);
            v[i + j] = hi, v[i + j + q] = lo;
          }
        }
      }
    }
  }
}

// The larger one; NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// One token on W lanes, by leading bits, for k <= KM.  Returns whether the next stage has to decide
// it (a comparison too close to call, or a NaN in the row); otherwise the slots are
// written when `write`.
template <typename T, int PER, int W, int KM>
__device__ __forceinline__ bool route_fast(const Args& a, int64_t t, bool write) {
  constexpr int SLOTS = (KM + W - 1) / W;
  constexpr int HEADS = PER < KM + 1 ? PER : KM + 1;  // words of a lane that k + 1 rounds can reach
  const float kLow = -INFINITY;
  const int lane = threadIdx.x & 31;
  const int li = lane & (W - 1);
  const int first_lane = lane & ~(W - 1);
  const uint32_t team = (W == 32 ? 0xffffffffu : ((1u << (W & 31)) - 1u)) << first_lane;
  const int group = li >> a.shift;
  const int in_group = (li & ((1 << a.shift) - 1)) * a.per;
  const int e0 = group * a.gs + in_group;
  const int n = group < a.G ? max(0, min(a.per, a.gs - in_group)) : 0;
  const T* row = static_cast<const T*>(a.logits) + t * a.E;
  const bool soft = a.score == MIRAI_SCORE_SOFTMAX;
  const bool scored = a.bias || (a.top2 && a.top_groups < a.G);  // scores take part in the choice

  float key[PER];
  load_row<PER>(row + e0, n, a.vec, key);
  float mx = kLow;
#pragma unroll
  for (int i = 0; i < PER; ++i) mx = max_nan(mx, key[i]);
  bool close = mx != mx;
  float smax = 1.f, inv = 1.f;
  float best1 = kLow, best2 = kLow;
  if (soft) {
    mx = max_lanes<W>(mx);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) sum += key[i] == kLow ? 0.f : ex2((key[i] - mx) * kLog2e);
    sum = sum_lanes<W>(sum);
    inv = sum == 0.f ? 0.f : 1.f / sum;
    smax = inv;
  }
  if (scored) {
    float bias[PER];
    if (a.bias) load_row<PER>(a.bias + e0, n, a.vec_bias, bias);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const bool open = key[i] != kLow;
      float v = soft ? ex2((key[i] - mx) * kLog2e) * inv : rcp(1.f + ex2(key[i] * -kLog2e));
      if (a.bias) {
        v = open ? v + bias[i] : kLow;
        v = fmaxf(v, kLow);  // (a NaN bias closes its expert)
        key[i] = v;
      } else {
        v = open ? v : kLow;
      }
      best2 = fmaxf(best2, fminf(best1, v));
      best1 = fmaxf(best1, v);
    }
  }
  if (!a.top2) {
    best1 = kLow;
#pragma unroll
    for (int i = 0; i < PER; ++i) best1 = fmaxf(best1, key[i]);
  }
  // Error of a score: ex2 and rcp are within 2^-22 of their values and the exponent's product
  // adds |x| 2^-24, times s (1 - s) <= 1/4 (and <= 0.23 / |x|), with two roundings of s: below
  // 2^-21.9 for sigmoid.  A softmax's terms add the rounding of their arguments (2^-18.5 at 87, below which
  // they are 0), their sum a few units more: below 2^-17 of the score, so of the largest.
  const float score_err = smax * (soft ? 0x1p-17f : 0x1.8p-22f);
  bool stays = group < a.G;
  if (a.top_groups < a.G) {
    for (int o = 1 << a.shift >> 1; o > 0; o >>= 1) {
      const float o1 = __shfl_xor_sync(0xffffffffu, best1, o), o2 = __shfl_xor_sync(0xffffffffu, best2, o);
      best2 = fmaxf(fmaxf(best2, o2), fminf(best1, o1));
      best1 = fmaxf(best1, o1);
    }
    const float gv = a.top2 && best2 != kLow ? best1 + best2 : best1;
    int rank = 0;
    for (int g = 0; g < a.G; ++g) {
      const float v = __shfl_sync(0xffffffffu, gv, first_lane + (g << a.shift));
      rank += v > gv || (v == gv && g < group);
    }
    stays = stays && rank < a.top_groups;
    if (scored) {
      const uint32_t in = __ballot_sync(0xffffffffu, group < a.G && rank == a.top_groups - 1) & team;
      const uint32_t out = __ballot_sync(0xffffffffu, group < a.G && rank == a.top_groups) & team;
      const float worst_in = __shfl_sync(0xffffffffu, gv, __ffs(in) - 1);
      const float best_out = __shfl_sync(0xffffffffu, gv, __ffs(out) - 1);
      // Every group has to keep clear of the middle by its own error: its scores', and the roundings of
      // s + bias and of their sum, which are as large as the addends (a sum near 0 of large ones is not).
      const bool two = a.top2 && best2 != kLow;
      const float err = 2.f * score_err + 0x1p-22f * (fabsf(best1) + (two ? fabsf(best2) : 0.f) + smax);
      const float mid = 0.5f * worst_in + 0.5f * best_out;
      if (best_out != kLow && group < a.G && gv != kLow)
        close |= !(rank < a.top_groups ? gv - mid > err : mid - gv > err);
    }
  }
  // leading bits of the key, then the id (lowest first), 0 for a closed slot
  const uint32_t ids = (1u << a.id_bits) - 1u;
  uint32_t v[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) v[i] = i < n && stays ? (order(key[i]) & ~ids) | (ids - (uint32_t)(e0 + i)) : 0u;
  sort_desc<PER>(v);
  int slot[SLOTS];
#pragma unroll
  for (int m = 0; m < SLOTS; ++m) slot[m] = 0;
  uint32_t last = 0;  // the word of slot k - 1, then the first one left out
  for (int j = 0; j <= a.k; ++j) {
    const uint32_t top = max_lanes<W>(v[0]);
    if (j == a.k) {
      // The cut: one word stands for every key left out, so equal (or, with the keys' errors,
      // too near) leading bits leave it open, unless they are the whole keys.  Among -inf the id decides.
      const uint32_t up = top | ids, above = last & ~ids;
      if (top && up != 0x007fffffu) {
        const float lo = __uint_as_float(above & 0x80000000u ? above & 0x7fffffffu : ~above);
        const float x = __uint_as_float(up & 0x80000000u ? up & 0x7fffffffu : ~up);
        bool tied = up >= above;
        // Logits as keys whose low bits are 0 (bf16 ones, or fp32 ones that were bf16) are ranked whole: a
        // tie, and the id has decided it.  They are common there: sent on, they cost [65536, 128]
        // in 8 groups 14 us more than 33, [65536, 256] 28 more than 64, in one group 43 more than 55.
        if (sizeof(T) == 2) {
          tied = tied && a.bias;
        } else if (!a.bias && tied) {  // (rare enough for fp32 logits to read the row again: a share per lane)
          uint32_t low = 0;
          for (int c = li; c < a.E; c += W) low |= __float_as_uint(load_logit(row + c));
          tied = (low & ids) != 0;
        }
        close |= tied || (a.bias && lo - x <= 2.f * score_err + 0x1p-22f * fabsf(x));
      }
      break;
    }
    last = top;
#pragma unroll
    for (int m = 0; m < SLOTS; ++m)
      if (j == m * W + li) slot[m] = (int)(ids - (top & ids));
    const bool pop = v[0] == top;
#pragma unroll
    for (int i = 0; i + 1 < HEADS; ++i) v[i] = pop ? v[i + 1] : v[i];
    v[HEADS - 1] = pop ? 0u : v[HEADS - 1];
  }
  // The slots' scores again, from their logits; their order by the whole key.
  float s[SLOTS], full[SLOTS], total = 0.f;
#pragma unroll
  for (int m = 0; m < SLOTS; ++m) {
    s[m] = 0.f;
    full[m] = kLow;
    if (m * W + li < a.k) {
      const float x = load_logit(row + slot[m]);
      if (x == x && x != kLow) {
        s[m] = soft ? expf(x - mx) * inv : 1.f / (1.f + expf(-x));
        full[m] = a.bias ? fmaxf(s[m] + __ldg(a.bias + slot[m]), kLow) : x;
      }
    }
    total += s[m];
  }
#pragma unroll
  for (int m = 0; m < SLOTS; ++m) {
    // the slot after this one: the next lane's, or the first lane's next
    const float same = __shfl_sync(0xffffffffu, full[m], first_lane + ((li + 1) & (W - 1)));
    const float wrap = __shfl_sync(0xffffffffu, full[m + 1 < SLOTS ? m + 1 : m], first_lane);
    const int id_same = __shfl_sync(0xffffffffu, slot[m], first_lane + ((li + 1) & (W - 1)));
    const int id_wrap = __shfl_sync(0xffffffffu, slot[m + 1 < SLOTS ? m + 1 : m], first_lane);
    const float next = li + 1 < W ? same : wrap;
    const int id = li + 1 < W ? id_same : id_wrap;
    if (m * W + li + 1 < a.k && next != kLow) {
      if (a.bias) close |= full[m] - next <= 2.f * score_err + 0x1p-22f * fabsf(next);
      else close |= next > full[m] || (next == full[m] && id < slot[m]);
    }
  }
  close = (__ballot_sync(0xffffffffu, close) & team) != 0;  // (no early return: shuffles take the whole warp)
  total = sum_lanes<W>(total);
  float den, scale;
  bool follows;
  denominator(a.norm, a.k, a.scale, total, den, scale, follows);
#pragma unroll
  for (int m = 0; m < SLOTS; ++m) {
    const int j = m * W + li;
    if (j >= a.k || !write || close) continue;
    a.idx[t * a.k + j] = slot[m];
    a.w[t * a.k + j] = s[m] / den * scale;
  }
  return close;
}

// One token on the whole warp, in 64 bits.
template <typename T, int PER>
__device__ __forceinline__ void route_exact(const Args& a, int64_t t) {
  using O = uint64_t;
  const double kLow = -INFINITY;
  const int lane = threadIdx.x & 31;
  const int group = lane >> a.shift32;
  const int in_group = (lane & ((1 << a.shift32) - 1)) * a.per32;
  const int e0 = group * a.gs + in_group;
  const int n = group < a.G ? max(0, min(a.per32, a.gs - in_group)) : 0;
  const T* row = static_cast<const T*>(a.logits) + t * a.E + e0;

  double key[PER], sc[PER];  // ranking key (-inf: closed by its logit) and score
  double mx = kLow;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const double l = i < n ? (double)load_logit(row + i) : kLow;
    nan |= l != l;
    key[i] = l != l ? kLow : l;
    mx = key[i] > mx ? key[i] : mx;
  }
  nan = __any_sync(0xffffffffu, nan);
  if (a.score == MIRAI_SCORE_SOFTMAX) {
    mx = max_lanes<32>(mx);
    double sum = 0.;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      sc[i] = key[i] == kLow ? 0. : exp(key[i] - mx);
      sum += sc[i];
    }
    sum = sum_lanes<32>(sum);
#pragma unroll
    for (int i = 0; i < PER; ++i) sc[i] = sum == 0. ? 0. : sc[i] / sum;
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) sc[i] = key[i] == kLow ? 0. : 1. / (1. + exp(-key[i]));
  }
  // group scores; without a bias they compare the scores' sums, or the logits
  double best1 = kLow, best2 = kLow;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const bool open = key[i] != kLow;
    if (a.bias) {
      key[i] = open ? sc[i] + (double)(i < n ? __ldg(a.bias + e0 + i) : 0.f) : kLow;
      if (key[i] != key[i]) key[i] = kLow;
    }
    const double v = a.top2 ? (open ? (a.bias ? key[i] : sc[i]) : kLow) : key[i];
    if (v > best1) best2 = best1, best1 = v;
    else if (v > best2) best2 = v;
  }
  bool stays = group < a.G;  // this lane's group is among the best
  if (a.top_groups < a.G) {
    for (int o = 1 << a.shift32 >> 1; o > 0; o >>= 1) {
      const double o1 = __shfl_xor_sync(0xffffffffu, best1, o), o2 = __shfl_xor_sync(0xffffffffu, best2, o);
      const double low = best1 < o1 ? best1 : o1;
      best1 = best1 < o1 ? o1 : best1;
      best2 = best2 < o2 ? o2 : best2;
      best2 = best2 < low ? low : best2;
    }
    const double gv = a.top2 && best2 != kLow ? best1 + best2 : best1;
    int rank = 0;
    for (int g = 0; g < a.G; ++g) {
      const double v = __shfl_sync(0xffffffffu, gv, g << a.shift32);
      rank += v > gv || (v == gv && g < group);
    }
    stays = stays && rank < a.top_groups;
  }
  // top-k: every lane offers its best key; the lowest of the best lanes wins
  uint64_t open_mask = stays && n > 0 ? ~0ull >> (64 - n) : 0ull;
  O best = 0;
  int best_i = 0;
  double best_s = 0.;
  auto rescan = [&]() {
    best = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const O o = (open_mask >> i) & 1u ? order(key[i]) : O(0);
      if (o > best) best = o, best_i = i, best_s = sc[i];
    }
  };
  rescan();
  int slot_e = 0;  // lane j: slot j
  double slot_s = 0., total = 0.;
  for (int j = 0; j < a.k; ++j) {
    const O top = max_lanes<32>(best);
    const int winner = __ffs(__ballot_sync(0xffffffffu, best == top)) - 1;
    const int e = __shfl_sync(0xffffffffu, e0 + best_i, winner);
    const double s = __shfl_sync(0xffffffffu, best_s, winner);
    total += s;
    if (j == lane) slot_e = e, slot_s = s;
    if (lane == winner) {
      open_mask &= ~(1ull << best_i);
      rescan();
    }
  }
  double den, scale;
  bool follows;
  denominator(a.norm, a.k, a.scale, total, den, scale, follows);
  if (lane < a.k) {
    a.idx[t * a.k + lane] = slot_e;
    a.w[t * a.k + lane] = nan ? __uint_as_float(0x7fffffffu) : (float)(slot_s / den * scale);
  }
}

// The warp's rows in `rows` (bit = first lane of the row's team), one after the other
// (kept out of the fast path's registers).
template <typename T, int PER, int W>
__device__ __noinline__ void route_exact_rows(const Args& a, int64_t first, uint32_t rows) {
  for (; rows; rows &= rows - 1) route_exact<T, PER>(a, first + (__ffs(rows) - 1) / W);
}

template <typename T, int PER, int W, int KM>
__global__ void __launch_bounds__(256, PER <= 16 ? 4 : (PER <= 32 ? 2 : 1))
    route_groups_kernel(const __grid_constant__ Args a) {
  constexpr int PER32 = W < 32 ? 4 : PER;  // experts per lane of a whole warp
  const int64_t t = ((int64_t)blockIdx.x * 256 + threadIdx.x) / W;
  const bool live = t < a.T;
  bool open = true;
  if constexpr (PER <= 32) open = route_fast<T, PER, W, KM>(a, live ? t : a.T - 1, live);  // past the end: unwritten
  const int lane = threadIdx.x & 31;
  const uint32_t rows = __ballot_sync(0xffffffffu, open && live && (lane & (W - 1)) == 0);
  if (rows) route_exact_rows<T, PER32, W>(a, t - lane / W, rows);
}

// ----------------------------------------------------------------------------
// Backward: dL/ds_j = scale a_j / den, a_j = g_j, or where den follows the scores' sum
// (den = sum + eps)  a_j = g_j - sum_i g_i s_i / den = sum_i (g_j - g_i) s_i / den + g_j eps / den;
//   sigmoid  dl_e = ds_e s (1 - s) at the selected experts, 0 elsewhere
//   softmax  dl_e = s_e (ds_e - sum_j ds_j s_j), the sum being scale sum_j g_j s_j / den, times
//            eps / den where den follows
// One score near 1 (a sure router) leaves nothing of a difference of rounded scores, so none is
// formed: 1 - s is the sigmoid of -l, or the other experts' share of the softmax, a_j is summed from
// differences of the gradients, and ds_e - sum_j ds_j s_j (den fixed) is g_e (1 - s_e) less the others' g s.
// W lanes per token (a warp takes 32 / W, since one token's chain of dependent loads is
// latency): the row is streamed once (softmax) and its gradient written once, zeros or the
// softmax tail everywhere, then slot j's lane corrects its expert (an index given twice
// gets the sum of both).  Lanes take vectors of four in turn, so rows move whole.
__device__ __forceinline__ void store_grad(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_grad(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void store4(float* p, const float* v) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void store4(__nv_bfloat16* p, const float* v) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
}

template <typename T, int PER, int W>
__global__ void __launch_bounds__(256) route_groups_backward_kernel(const float* __restrict__ grad_w,
                                                                    const T* __restrict__ logits,
                                                                    const int64_t* __restrict__ idx, int64_t tokens,
                                                                    int E, int k, int score, int norm, int vec,
                                                                    float route_scale, T* __restrict__ out) {
  constexpr int SLOTS = (kMaxTopK + W - 1) / W;
  const int lane = threadIdx.x & 31, li = lane & (W - 1);
  const int64_t own = ((int64_t)blockIdx.x * 256 + threadIdx.x) / W;
  const bool live = own < tokens;
  const int64_t t = live ? own : tokens - 1;  // lanes past the end repeat the last token, unwritten
  const T* row = logits + t * E;
  T* grow = out + t * E;
  const bool soft = score == MIRAI_SCORE_SOFTMAX;
  // the slots' ids and gradients first: their logits hang on them
  int e[SLOTS];
  float g[SLOTS], s[SLOTS], x[SLOTS];
#pragma unroll
  for (int m = 0; m < SLOTS; ++m) {
    const int j = m * W + li;
    e[m] = -1;
    g[m] = x[m] = 0.f;
    if (j < k) {
      const int64_t id = idx[t * k + j];
      g[m] = grad_w[t * k + j];
      if (id < 0 || id >= E) {
        if (live) device_fail(MIRAI_ERR_DEVICE_BOUNDS, 750);
      } else {
        e[m] = (int)id;
        x[m] = load_logit(row + id);
      }
    }
  }
  float l[PER];
  float mx = -INFINITY, inv = 0.f;
  float others = 0.f;  // softmax: what the largest score leaves of 1
  if (soft) {
#pragma unroll
    for (int i = 0; i < PER; i += 4) {
      const int c = (i / 4 * W + li) * 4;
      float v[4];
      load_row<4>(row + c, E - c, vec, v);
#pragma unroll
      for (int z = 0; z < 4; ++z) l[i + z] = v[z], mx = fmaxf(mx, v[z]);
    }
    mx = max_lanes<W>(mx);
    float most = 0.f, rest = 0.f;  // the terms at the maximum (each 1, or NaN), and below it
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const bool at = l[i] == mx;
      l[i] = l[i] == -INFINITY ? 0.f : ex2((l[i] - mx) * kLog2e);  // from here on: the scores
      most += at ? l[i] : 0.f;
      rest += at ? 0.f : l[i];
    }
    most = sum_lanes<W>(most);
    rest = sum_lanes<W>(rest);
    const float sum = most + rest;
    inv = sum == 0.f ? 0.f : 1.f / sum;
    others = (rest + (most - 1.f)) * inv;
  }
  float total = 0.f, left[SLOTS];  // left: 1 - s
#pragma unroll
  for (int m = 0; m < SLOTS; ++m) {
    s[m] = e[m] < 0 || x[m] == -INFINITY ? 0.f : (soft ? expf(x[m] - mx) * inv : 1.f / (1.f + expf(-x[m])));
    left[m] = !soft ? 1.f / (1.f + expf(x[m])) : (x[m] == mx ? others : 1.f - s[m]);  // (below the maximum: s <= 1/2)
    total += s[m];
  }
  float den, scale;
  bool follows;
  denominator(norm, k, route_scale, sum_lanes<W>(total), den, scale, follows);
  const float eps_den = follows && norm == MIRAI_NORM_EPS ? 1e-20f / den : 0.f;
  float mean = 0.f, share[SLOTS];
#pragma unroll
  for (int m = 0; m < SLOTS; ++m) {
    share[m] = s[m] / den;
    if (e[m] >= 0) mean += g[m] * share[m];
  }
  mean = sum_lanes<W>(mean);
  const float dot = scale * mean * (follows ? eps_den : 1.f);  // sum_j ds_j s_j
  // Every pair of slots: a_j, and whether an expert is named twice.  (By the whole warp: the
  // tokens of one may differ in `follows`.)
  float a[SLOTS];
  bool twice = false;
#pragma unroll
  for (int m = 0; m < SLOTS; ++m) a[m] = follows ? g[m] * eps_den : 0.f;
#pragma unroll
  for (int m2 = 0; m2 < SLOTS; ++m2) {
    for (int j = 0; j < W && m2 * W + j < k; ++j) {
      const int from = (lane & ~(W - 1)) + j;
      const int other = __shfl_sync(0xffffffffu, e[m2], from);
      const float go = __shfl_sync(0xffffffffu, g[m2], from);
      const float so = __shfl_sync(0xffffffffu, follows ? share[m2] : s[m2], from);
#pragma unroll
      for (int m = 0; m < SLOTS; ++m) {
        const bool same = other == e[m];
        if (follows) {
          a[m] = fmaf(g[m] - go, so, a[m]);
          twice |= same && e[m] >= 0 && (m2 != m || j != li);
        } else if (same) {  // (den fixed: a slot already holds its expert's sum)
          a[m] = fmaf(go, soft ? left[m] : 1.f, a[m]);
        } else if (soft) {
          a[m] = fmaf(-go, so, a[m]);
        }
      }
    }
  }
  if (__any_sync(0xffffffffu, twice)) {  // slots that name the same expert share the sum of theirs
    float sums[SLOTS];
#pragma unroll
    for (int m = 0; m < SLOTS; ++m) sums[m] = 0.f;
#pragma unroll
    for (int m2 = 0; m2 < SLOTS; ++m2) {
      for (int j = 0; j < W && m2 * W + j < k; ++j) {
        const int other = __shfl_sync(0xffffffffu, e[m2], (lane & ~(W - 1)) + j);
        const float v = __shfl_sync(0xffffffffu, a[m2], (lane & ~(W - 1)) + j);
#pragma unroll
        for (int m = 0; m < SLOTS; ++m)
          if (other == e[m]) sums[m] += v;
      }
    }
#pragma unroll
    for (int m = 0; m < SLOTS; ++m) a[m] = follows ? sums[m] : a[m];
  }
  const float tail = -inv * dot;
  if (live) {
#pragma unroll
    for (int i = 0; i < PER; i += 4) {
      const int c = (i / 4 * W + li) * 4;
      float v[4];
#pragma unroll
      for (int z = 0; z < 4; ++z) v[z] = soft ? l[i + z] * tail : 0.f;
      if (vec) {
        if (c < E) store4(grow + c, v);
      } else {
#pragma unroll
        for (int z = 0; z < 4; ++z)
          if (c + z < E) store_grad(grow + c + z, v[z]);
      }
    }
  }
  __syncwarp();
  if (live) {
#pragma unroll
    for (int m = 0; m < SLOTS; ++m)
      if (e[m] >= 0) {
        // den fixed, softmax: a is ds_e - sum_j ds_j s_j already (times den / scale)
        const float d = scale * share[m] * a[m];
        store_grad(grow + e[m], !soft ? d * left[m] : (follows ? d - s[m] * dot : d));
      }
  }
}

static int route_problem(const char* name, int64_t T, int32_t E, int32_t k, int32_t score, int32_t norm, int32_t dtype) {
  if (T < 0 || E <= 0 || E > kMaxExperts)
    return set_error(MIRAI_ERR_INVALID_ARG, "%s: bad sizes (T=%lld, E=%d, 1..%d experts)", name, (long long)T, E,
                     kMaxExperts);
  if (k <= 0 || k > E || k > kMaxTopK)
    return set_error(MIRAI_ERR_INVALID_ARG, "%s: needs 1 <= k <= min(E, %d) (k=%d, E=%d)", name, kMaxTopK, k, E);
  if (score != MIRAI_SCORE_SOFTMAX && score != MIRAI_SCORE_SIGMOID)
    return set_error(MIRAI_ERR_INVALID_ARG, "%s: unknown score function %d", name, score);
  if (norm < MIRAI_NORM_NONE || norm > MIRAI_NORM_L1)
    return set_error(MIRAI_ERR_INVALID_ARG, "%s: unknown normalisation %d", name, norm);
  if (dtype != MIRAI_DTYPE_F32 && dtype != MIRAI_DTYPE_BF16)
    return set_error(MIRAI_ERR_INVALID_ARG, "%s: logits must be fp32 or bf16 (dtype %d)", name, dtype);
  if (T > (int64_t)INT32_MAX * 8)
    return set_error(MIRAI_ERR_UNSUPPORTED, "%s: too many tokens for one call", name);
  return MIRAI_OK;
}

template <typename T, int PER, int W> static void launch(const Args& a, cudaStream_t s) {
  const unsigned grid = (unsigned)((a.T * W + 255) / 256);
  if constexpr (PER <= 8) {
    if (a.k <= 8) {
      route_groups_kernel<T, PER, W, 8><<<grid, 256, 0, s>>>(a);
      return;
    }
  }
  route_groups_kernel<T, PER, W, kMaxTopK><<<grid, 256, 0, s>>>(a);
}

template <typename T> static int dispatch(Args a, cudaStream_t s) {
  a.id_bits = 1;
  while ((1 << a.id_bits) < a.E) ++a.id_bits;
  // The fewest lanes per token that keep a group on whole lanes and 8 experts a lane.  (16 a lane, and
  // half the lanes, measured 48 against 46 us for [65536, 128], 33 against 34 for [21847, 256].)
  int W = 8;
  for (;; W *= 2) {
    if (W < a.G) continue;
    a.shift = 0;
    while ((2 << a.shift) * a.G <= W) ++a.shift;
    a.per = (a.gs + (1 << a.shift) - 1) >> a.shift;
    if (a.per <= 8 || W == 32) break;
  }
  a.shift32 = 0;
  while ((2 << a.shift32) * a.G <= 32) ++a.shift32;
  a.per32 = (a.gs + (1 << a.shift32) - 1) >> a.shift32;  // <= 4 where W < 32: 8 experts a lane, 2 or 4 times the lanes
  const bool vec = a.E % 4 == 0 && a.gs % 4 == 0 && a.per % 4 == 0;
  a.vec = vec && (reinterpret_cast<uintptr_t>(a.logits) & 15) == 0;
  a.vec_bias = vec && (reinterpret_cast<uintptr_t>(a.bias) & 15) == 0;
  if (W == 8) launch<T, 8, 8>(a, s);
  else if (W == 16) launch<T, 8, 16>(a, s);
  else if (a.per <= 8) launch<T, 8, 32>(a, s);
  else if (a.per <= 16) launch<T, 16, 32>(a, s);
  else if (a.per <= 32) launch<T, 32, 32>(a, s);
  else launch<T, 64, 32>(a, s);  // a.per <= 64: see route_groups
  return check_launch("route_groups");
}

template <typename T, int PER, int W>
static void backward(const float* gw, const void* logits, const int64_t* idx, int64_t tokens, int E, int k, int score,
                     int norm, float scale, void* out, cudaStream_t s) {
  const int vec = E % 4 == 0 && ((reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(out)) & 15) == 0;
  route_groups_backward_kernel<T, PER, W><<<(unsigned)((tokens * W + 255) / 256), 256, 0, s>>>(
      gw, static_cast<const T*>(logits), idx, tokens, E, k, score, norm, vec, scale, static_cast<T*>(out));
}

template <typename T>
static void launch_backward(const float* gw, const void* logits, const int64_t* idx, int64_t tokens, int E, int k,
                            int score, int norm, float scale, void* out, cudaStream_t s) {
  if (E <= 64) backward<T, 8, 8>(gw, logits, idx, tokens, E, k, score, norm, scale, out, s);
  else if (E <= 128) backward<T, 16, 8>(gw, logits, idx, tokens, E, k, score, norm, scale, out, s);
  else if (E <= 256) backward<T, 16, 16>(gw, logits, idx, tokens, E, k, score, norm, scale, out, s);
  else backward<T, 32, 32>(gw, logits, idx, tokens, E, k, score, norm, scale, out, s);
}

}  // namespace rg
}  // namespace mirai

using namespace mirai;

extern "C" {

int mirai_route_groups(const void* logits, int32_t logits_dtype, int64_t num_tokens, int32_t num_experts, int32_t top_k,
                       int32_t num_groups, int32_t top_groups, int32_t group_top2, int32_t score_func,
                       const float* choice_bias, int32_t norm_mode, float route_scale, int64_t* top_indices,
                       float* top_weights, mirai_stream_t stream) {
  if (int rc = rg::route_problem("route_groups", num_tokens, num_experts, top_k, score_func, norm_mode, logits_dtype))
    return rc;
  if (num_groups <= 0 || num_groups > rg::kMaxGroups || num_experts % num_groups)
    return set_error(MIRAI_ERR_INVALID_ARG, "route_groups: %d experts in %d groups (1..%d groups of one size)",
                     num_experts, num_groups, rg::kMaxGroups);
  const int gs = num_experts / num_groups;
  if (top_groups <= 0 || top_groups > num_groups || top_groups * gs < top_k)
    return set_error(MIRAI_ERR_INVALID_ARG, "route_groups: %d of %d groups of %d experts for k=%d", top_groups, num_groups,
                     gs, top_k);
  if (num_tokens == 0) return MIRAI_OK;
  if (!logits || !top_indices || !top_weights) return set_error(MIRAI_ERR_INVALID_ARG, "route_groups: null pointer");
  rg::Args a = {};
  a.logits = logits;
  a.bias = choice_bias;
  a.T = num_tokens;
  a.E = num_experts;
  a.k = top_k;
  a.G = num_groups;
  a.top_groups = top_groups;
  a.gs = gs;
  a.score = score_func;
  a.top2 = group_top2 && gs > 1;
  a.norm = norm_mode;
  a.scale = route_scale;
  a.idx = top_indices;
  a.w = top_weights;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return logits_dtype == MIRAI_DTYPE_F32 ? rg::dispatch<float>(a, s) : rg::dispatch<__nv_bfloat16>(a, s);
}

int mirai_route_groups_backward(const float* grad_weights, const void* logits, int32_t logits_dtype,
                                const int64_t* top_indices, int64_t num_tokens, int32_t num_experts, int32_t top_k,
                                int32_t score_func, int32_t norm_mode, float route_scale, void* grad_logits,
                                mirai_stream_t stream) {
  if (int rc = rg::route_problem("route_groups_backward", num_tokens, num_experts, top_k, score_func, norm_mode,
                                 logits_dtype))
    return rc;
  if (num_tokens == 0) return MIRAI_OK;
  if (!grad_weights || !logits || !top_indices || !grad_logits)
    return set_error(MIRAI_ERR_INVALID_ARG, "route_groups_backward: null pointer");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (logits_dtype == MIRAI_DTYPE_F32)
    rg::launch_backward<float>(grad_weights, logits, top_indices, num_tokens, num_experts, top_k, score_func, norm_mode,
                               route_scale, grad_logits, s);
  else
    rg::launch_backward<__nv_bfloat16>(grad_weights, logits, top_indices, num_tokens, num_experts, top_k, score_func,
                                       norm_mode, route_scale, grad_logits, s);
  return check_launch("route_groups_backward");
}

}  // extern "C"
