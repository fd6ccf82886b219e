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
// it (about one in a thousand) is decided again in 64 bits by the same code.
// Without a bias, experts and group maxima are ranked by the logits themselves,
// which is exact.
//
// W lanes hold a token's experts, so a warp routes 32 / W tokens: each group on
// whole lanes (a power of two of them), PER experts per lane, so that expert
// order is lane order, group scores are butterflies inside a group, and ties
// resolve to the lowest lane.
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
  int score;    // MIRAI_SCORE_*
  int top2;     // group score: 1 the two best scores, 0 the best key
  int norm;     // MIRAI_NORM_*
  float scale;
  int64_t* idx;
  float* w;
};

__device__ __forceinline__ float load_logit(const float* p) { return __ldg(p); }
__device__ __forceinline__ float load_logit(const __nv_bfloat16* p) { return __bfloat162float(*p); }

__device__ __forceinline__ float real_exp(float x) { return expf(x); }
__device__ __forceinline__ double real_exp(double x) { return exp(x); }

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
    const V x = __shfl_xor_sync(0xffffffffu, v, o);
    v = x > v ? x : v;
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

// One token on W lanes.  Returns (fp32 only) whether a comparison was too close
// to call; otherwise, and always in 64 bits, its slots are written when `write`.
template <typename F, typename T, int PER, int W>
__device__ __forceinline__ bool route_row(const Args& a, int64_t t, bool write) {
  constexpr bool FAST = sizeof(F) == 4;
  constexpr int SLOTS = (kMaxTopK + W - 1) / W;
  const F kLow = -INFINITY;
  const int lane = threadIdx.x & 31;
  const int li = lane & (W - 1);
  const int first_lane = lane & ~(W - 1);
  const uint32_t team = (W == 32 ? 0xffffffffu : ((1u << (W & 31)) - 1u)) << first_lane;
  const int group = li >> a.shift;
  const int in_group = (li & ((1 << a.shift) - 1)) * a.per;
  const int e0 = group * a.gs + in_group;
  const int n = group < a.G ? max(0, min(a.per, a.gs - in_group)) : 0;
  const T* row = static_cast<const T*>(a.logits) + t * a.E + e0;

  F key[PER], sc[PER];  // ranking key (-inf: closed by its logit) and score
  F mx = kLow;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const F l = i < n ? F(load_logit(row + i)) : kLow;
    nan |= l != l;
    key[i] = l != l ? kLow : l;
    mx = key[i] > mx ? key[i] : mx;
  }
  nan = (__ballot_sync(0xffffffffu, nan) & team) != 0;
  F smax = F(1);  // bounds every score
  if (a.score == MIRAI_SCORE_SOFTMAX) {
    mx = max_lanes<W>(mx);
    F sum = F(0);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      sc[i] = key[i] == kLow ? F(0) : real_exp(key[i] - mx);
      sum += sc[i];
    }
    sum = sum_lanes<W>(sum);
    smax = sum == F(0) ? F(0) : F(1) / sum;
#pragma unroll
    for (int i = 0; i < PER; ++i) sc[i] *= smax;
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) sc[i] = key[i] == kLow ? F(0) : F(1) / (F(1) + real_exp(-key[i]));
  }
  // Error of a score: sigmoid within 4 roundings of a value <= 1; softmax within 70
  // (its sum) of a value <= smax.  A bias adds half a unit of the key.
  const F score_err = smax * (a.score == MIRAI_SCORE_SOFTMAX ? F(0x1p-17f) : F(0x1p-21f));
  bool close = false;

  // group scores; without a bias they compare the scores' sums, or the logits
  F best1 = kLow, best2 = kLow;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const bool open = key[i] != kLow;
    if (a.bias) {
      const F b = F(i < n ? __ldg(a.bias + e0 + i) : 0.f);
      key[i] = open ? sc[i] + b : kLow;
      if (key[i] != key[i]) key[i] = kLow;
    }
    const F v = a.top2 ? (open ? (a.bias ? key[i] : sc[i]) : kLow) : key[i];
    if (v > best1) best2 = best1, best1 = v;
    else if (v > best2) best2 = v;
  }
  bool stays = true;  // this lane's group is among the best
  if (a.top_groups < a.G) {
    for (int o = 1 << a.shift >> 1; o > 0; o >>= 1) {
      const F o1 = __shfl_xor_sync(0xffffffffu, best1, o), o2 = __shfl_xor_sync(0xffffffffu, best2, o);
      const F low = best1 < o1 ? best1 : o1;
      best1 = best1 < o1 ? o1 : best1;
      best2 = best2 < o2 ? o2 : best2;
      best2 = best2 < low ? low : best2;
    }
    const F gv = a.top2 && best2 != kLow ? best1 + best2 : best1;
    int rank = 0;
    for (int g = 0; g < a.G; ++g) {
      const F v = __shfl_sync(0xffffffffu, gv, first_lane + (g << a.shift));
      rank += v > gv || (v == gv && g < group);
    }
    stays = group < a.G && rank < a.top_groups;
    if (FAST && (a.top2 || a.bias)) {  // the last group in against the first one out
      const uint32_t in = __ballot_sync(0xffffffffu, group < a.G && rank == a.top_groups - 1) & team;
      const uint32_t out = __ballot_sync(0xffffffffu, group < a.G && rank == a.top_groups) & team;
      const F worst_in = __shfl_sync(0xffffffffu, gv, __ffs(in) - 1);
      const F best_out = __shfl_sync(0xffffffffu, gv, __ffs(out) - 1);
      if (best_out != kLow)
        close |= worst_in - best_out <= F(4) * score_err + F(0x1p-21f) * (fabs(worst_in) + fabs(best_out) + smax);
    }
  }

  // top-k: every lane offers its best key; the lowest of the best lanes wins
  using O = decltype(order(F(0)));
  uint32_t open_mask[(PER + 31) / 32];
#pragma unroll
  for (int m = 0; m < (PER + 31) / 32; ++m) open_mask[m] = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (i < n && stays) open_mask[i / 32] |= 1u << (i & 31);
  O best = 0;
  int best_i = 0;
  F best_s = F(0);
  auto rescan = [&]() {
    best = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const O o = (open_mask[i / 32] >> (i & 31)) & 1u ? order(key[i]) : O(0);
      if (o > best) best = o, best_i = i, best_s = sc[i];
    }
  };
  rescan();
  int slot_e[SLOTS];
  F slot_s[SLOTS];
#pragma unroll
  for (int m = 0; m < SLOTS; ++m) slot_e[m] = 0, slot_s[m] = F(0);
  F total = F(0), previous = INFINITY;
  const bool check = FAST && a.bias != nullptr;
  const F key_err = F(2) * score_err;
  for (int j = 0; j < a.k + (check ? 1 : 0); ++j) {
    const O top = max_lanes<W>(best);
    if (check) {
      const F v = __uint_as_float(top & 0x80000000u ? (uint32_t)top & 0x7fffffffu : ~(uint32_t)top);
      if (top && v != kLow) close |= previous - v <= key_err + F(0x1p-22f) * fabs(v);
      previous = v;
      if (j == a.k) break;
    }
    const uint32_t who = __ballot_sync(0xffffffffu, best == top) & team;
    const int winner = __ffs(who) - 1;
    const int e = __shfl_sync(0xffffffffu, e0 + best_i, winner);
    const F s = __shfl_sync(0xffffffffu, best_s, winner);
    total += s;
#pragma unroll
    for (int m = 0; m < SLOTS; ++m)
      if (j == m * W + li) slot_e[m] = e, slot_s[m] = s;
    if (lane == winner) {
#pragma unroll
      for (int m = 0; m < (PER + 31) / 32; ++m)
        if (best_i / 32 == m) open_mask[m] &= ~(1u << (best_i & 31));
      rescan();
    }
  }
  if (FAST && (__ballot_sync(0xffffffffu, close) & team)) return true;
  if (!write) return false;
  F den, scale;
  bool follows;
  denominator(a.norm, a.k, a.scale, total, den, scale, follows);
#pragma unroll
  for (int m = 0; m < SLOTS; ++m) {
    const int j = m * W + li;
    if (j >= a.k) continue;
    a.idx[t * a.k + j] = slot_e[m];
    a.w[t * a.k + j] = nan ? __uint_as_float(0x7fffffffu) : (float)(slot_s[m] / den * scale);
  }
  return false;
}

// The rows of a warp that fp32 could not decide, in 64 bits (rare: kept out of the fast path's registers).
template <typename T, int PER, int W> __device__ __noinline__ void route_close_rows(const Args& a, int64_t t, bool write) {
  route_row<double, T, PER, W>(a, t, write);
}

template <typename T, int PER, int W> __global__ void __launch_bounds__(256) route_groups_kernel(const __grid_constant__ Args a) {
  const int64_t t = ((int64_t)blockIdx.x * 256 + threadIdx.x) / W;
  const bool live = t < a.T;
  const int64_t tc = live ? t : a.T - 1;  // lanes past the end repeat the last token, unwritten
  const bool close = route_row<float, T, PER, W>(a, tc, live);
  if (__any_sync(0xffffffffu, close)) route_close_rows<T, PER, W>(a, tc, live && close);
}

// ----------------------------------------------------------------------------
// Backward: dL/ds_j = scale (g_j - [den follows] sum_i g_i s_i / den) / den, then
//   sigmoid  dl_e = ds s (1 - s) at the selected experts, 0 elsewhere
//   softmax  dl_e = s_e (ds_e - sum_j ds_j s_j)
// One warp per token: the row is streamed once (softmax) and its gradient
// written once, zeros or the softmax tail everywhere, then lane j corrects slot j's
// expert (an index given twice gets the sum of both).
__device__ __forceinline__ void store_grad(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_grad(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

template <typename T, int PER>
__global__ void __launch_bounds__(256) route_groups_backward_kernel(const float* __restrict__ grad_w,
                                                                    const T* __restrict__ logits,
                                                                    const int64_t* __restrict__ idx, int64_t tokens,
                                                                    int E, int k, int score, int norm,
                                                                    float route_scale, T* __restrict__ out) {
  const int lane = threadIdx.x & 31;
  const int64_t t = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (t >= tokens) return;
  const T* row = logits + t * E;
  T* grow = out + t * E;
  const bool soft = score == MIRAI_SCORE_SOFTMAX;
  float l[PER];
  float mx = -INFINITY, inv = 0.f;
  if (soft) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = i * 32 + lane;
      l[i] = e < E ? load_logit(row + e) : -INFINITY;
      mx = fmaxf(mx, l[i]);
    }
    mx = max_lanes<32>(mx);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      l[i] = l[i] == -INFINITY ? 0.f : expf(l[i] - mx);  // from here on: the scores
      sum += l[i];
    }
    sum = sum_lanes<32>(sum);
    inv = sum == 0.f ? 0.f : 1.f / sum;
  }
  int64_t e = -1;
  float s = 0.f, g = 0.f;
  if (lane < k) {
    e = idx[t * k + lane];
    if (e < 0 || e >= E) {
      device_fail(MIRAI_ERR_DEVICE_BOUNDS, 750);
      e = -1;
    } else {
      const float x = load_logit(row + e);
      s = x == -INFINITY ? 0.f : (soft ? expf(x - mx) * inv : 1.f / (1.f + expf(-x)));
      g = grad_w[t * k + lane];
    }
  }
  float den, scale;
  bool follows;
  denominator(norm, k, route_scale, sum_lanes<32>(s), den, scale, follows);
  const float mean = follows ? sum_lanes<32>(g * (s / den)) : 0.f;
  const float ds = e >= 0 ? scale * ((g - mean) / den) : 0.f;
  float mine = ds * s;  // this slot's share of dL/ds * s, and the same of slots that name its expert
  const float dot = sum_lanes<32>(mine);
  float sums = 0.f;
  for (int j = 0; j < k; ++j) {
    const int64_t other = __shfl_sync(0xffffffffu, e, j);
    const float v = __shfl_sync(0xffffffffu, mine, j);
    if (other == e) sums += v;
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int x = i * 32 + lane;
    if (x < E) store_grad(grow + x, soft ? -(l[i] * inv) * dot : 0.f);
  }
  __syncwarp();
  if (e >= 0) store_grad(grow + e, soft ? sums - s * dot : sums * (1.f - s));
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
  route_groups_kernel<T, PER, W><<<(unsigned)((a.T * W + 255) / 256), 256, 0, s>>>(a);
}

template <typename T> static int dispatch(Args a, cudaStream_t s) {
  // the fewest lanes per token that keep a group on whole lanes and 16 experts a lane
  int W = 8;
  for (;; W *= 2) {
    if (W < a.G) continue;
    a.shift = 0;
    while ((2 << a.shift) * a.G <= W) ++a.shift;
    a.per = (a.gs + (1 << a.shift) - 1) >> a.shift;
    if (a.per <= 16 || W == 32) break;
  }
  if (W == 8) a.per <= 8 ? launch<T, 8, 8>(a, s) : launch<T, 16, 8>(a, s);
  else if (W == 16) a.per <= 8 ? launch<T, 8, 16>(a, s) : launch<T, 16, 16>(a, s);
  else if (a.per <= 8) launch<T, 8, 32>(a, s);
  else if (a.per <= 16) launch<T, 16, 32>(a, s);
  else if (a.per <= 32) launch<T, 32, 32>(a, s);
  else launch<T, 64, 32>(a, s);  // a.per <= 64: see route_groups
  return check_launch("route_groups");
}

template <typename T>
static void launch_backward(const float* gw, const void* logits, const int64_t* idx, int64_t tokens, int E, int k,
                            int score, int norm, float scale, void* out, cudaStream_t s) {
  const unsigned grid = (unsigned)((tokens + 7) / 8);
  const T* l = static_cast<const T*>(logits);
  T* o = static_cast<T*>(out);
  if (E <= 128) route_groups_backward_kernel<T, 4><<<grid, 256, 0, s>>>(gw, l, idx, tokens, E, k, score, norm, scale, o);
  else if (E <= 256) route_groups_backward_kernel<T, 8><<<grid, 256, 0, s>>>(gw, l, idx, tokens, E, k, score, norm, scale, o);
  else route_groups_backward_kernel<T, 32><<<grid, 256, 0, s>>>(gw, l, idx, tokens, E, k, score, norm, scale, o);
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
