// Expert routing from router logits, and its gradient: one warp per token.
//
//   s = softmax(l) or sigmoid(l)          scores of the E experts
//   c = s + bias                          choices (bias: the balance bias)
//   group score = sum of the group's best two choices, or its best one;
//   the best topk_groups groups stay      (equal scores: lower group first)
//   idx = top-k of c among them           (equal choices: lower expert first)
//   w = s[idx], renormalised by max(sum, 1e-9) if asked for, times scale
//
// An expert whose logit or bias is -inf is masked: it ranks behind all others
// and its weight is 0, so a token whose mask leaves nothing gets the lowest
// expert ids with weights 0.  NaN ranks first, so that it is seen.
//
// Two choices can lie closer together than fp32 resolves them (at 256 experts
// about one token in 300), and which of them wins decides an index.  So the
// fp32 selection also looks at the gaps next to every decision it makes; a
// token with a gap inside the fp32 error is decided again from fp64 scores.
// Without a bias the choices are monotonic in the logits, which decide then,
// exactly.
#include "sb_common.cuh"
#include "sb_internal.h"

namespace sb {

constexpr int kRouteMaxE = 1024;
constexpr int kRouteMaxK = 32;
constexpr int kRouteMaxGroups = 32;

// Order-preserving integer of a float: NaN above +inf, -0 equal to +0; every
// value, -inf too, is above 0, which marks an expert that is not a candidate.
SB_DEVINL uint32_t order_key(float v) {
  if (v != v) return 0xffffffffu;
  const uint32_t u = __float_as_uint(v + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
SB_DEVINL unsigned long long order_key(double v) {
  if (v != v) return ~0ull;
  const unsigned long long u = static_cast<unsigned long long>(__double_as_longlong(v + 0.0));
  return (u >> 63) ? ~u : (u | (1ull << 63));
}
SB_DEVINL float key_value(uint32_t k) {
  if (k == 0xffffffffu) return __uint_as_float(0x7fc00000u);
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
SB_DEVINL double key_value(unsigned long long k) {
  if (k == ~0ull) return __longlong_as_double(0x7ff8000000000000ll);
  return __longlong_as_double(static_cast<long long>((k >> 63) ? (k & ~(1ull << 63)) : ~k));
}
SB_DEVINL uint32_t warp_max_key(uint32_t k) { return __reduce_max_sync(0xffffffffu, k); }
SB_DEVINL unsigned long long warp_max_key(unsigned long long k) {
  const uint32_t hi = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(k >> 32));
  const uint32_t lo = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(k >> 32) == hi ? static_cast<uint32_t>(k) : 0u);
  return (static_cast<unsigned long long>(hi) << 32) | lo;
}

struct RouteParams {
  int64_t ld;
  int n, E, K, score;
  const float* bias;
  int groups, topk_groups, group_top, renorm;
  float scale;
  int32_t* top_idx;
  float* top_w;
};

// Which of a token's candidates are taken.  key[v] is the order key of expert
// lane + 32 v (0: not a candidate); returns, in lane j < K, the j-th expert.
// With kCheck, *close is set when an expert was taken while another one that is
// not exactly equal to it (same logit, same bias) lay within the fp32 error.
template <int V, bool kCheck, typename Key>
SB_DEVINL int select_top(Key (&key)[V], const float (&l)[V], const float (&b)[V], int K, int lane, float tol,
                         bool* close) {
  int mine = 0;
  bool near = false;
  for (int j = 0; j < K; ++j) {
    Key best = key[0];
#pragma unroll
    for (int v = 1; v < V; ++v) best = key[v] > best ? key[v] : best;
    const Key top = warp_max_key(best);
    uint32_t e = 0xffffffffu;
#pragma unroll
    for (int v = V - 1; v >= 0; --v)
      if (key[v] == top) e = lane + 32 * v;
    e = __reduce_min_sync(0xffffffffu, e);
    if (kCheck) {
      float cl = 0.f, cb = 0.f;
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (lane + 32 * v == static_cast<int>(e)) { cl = l[v]; cb = b[v]; }
      cl = __shfl_sync(0xffffffffu, cl, e & 31);
      cb = __shfl_sync(0xffffffffu, cb, e & 31);
      const float c = static_cast<float>(key_value(top));
      const Key limit = order_key(c - (tol + fabsf(c) * 0x1p-22f));
#pragma unroll
      for (int v = 0; v < V; ++v) near |= key[v] >= limit && key[v] != 0 && (l[v] != cl || b[v] != cb);
    }
    if (lane == j) mine = static_cast<int>(e);
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (lane + 32 * v == static_cast<int>(e)) key[v] = 0;
  }
  if (kCheck) *close |= __any_sync(0xffffffffu, near);
  return mine;
}

// Drops the candidates outside the best topk_groups groups.  ch: the warp's
// keys of all experts in shared memory.
template <int V, bool kCheck, typename Key>
SB_DEVINL void keep_groups(Key (&key)[V], Key* ch, const RouteParams& p, int lane, float tol, bool* close) {
  using Val = decltype(key_value(Key(0)));
  const int per = p.E / p.groups;
#pragma unroll
  for (int v = 0; v < V; ++v)
    if (lane + 32 * v < p.E) ch[lane + 32 * v] = key[v];
  __syncwarp();
  Key gk = 0;
  if (lane < p.groups) {
    Key k1 = 0, k2 = 0;
    for (int i = 0; i < per; ++i) {
      const Key k = ch[lane * per + i];
      if (k > k1) { k2 = k1; k1 = k; } else if (k > k2) k2 = k;
    }
    Val gs = key_value(k1);
    if (p.group_top == 2 && per > 1) gs += key_value(k2);
    gk = order_key(gs);
  }
  __syncwarp();
  uint32_t kept = 0;
  Key top = 0;
  for (int j = 0; j < p.topk_groups; ++j) {
    top = warp_max_key(gk);
    const int g = __ffs(__ballot_sync(0xffffffffu, gk == top)) - 1;
    kept |= 1u << g;
    if (lane == g) gk = 0;
  }
  if (kCheck) {  // a group left out within the error of the last one kept
    const float c = static_cast<float>(key_value(top));
    *close |= __any_sync(0xffffffffu, gk != 0 && gk >= order_key(c - (2.f * tol + fabsf(c) * 0x1p-21f)));
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = lane + 32 * v;
    if (e < p.E && !((kept >> (e / per)) & 1u)) key[v] = 0;
  }
}

// The selection from fp64 scores.
template <int V>
__device__ __noinline__ int select_f64(const float (&l)[V], const float (&b)[V], const RouteParams& p,
                                       unsigned long long* ch, int lane) {
  double m = -INFINITY, sum = 0.0;
  if (p.score == SB_SCORE_SOFTMAX) {
    float mf = -INFINITY;
#pragma unroll
    for (int v = 0; v < V; ++v) mf = fmaxf(mf, l[v]);
    m = warp_max(mf);
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (l[v] > -INFINITY) sum += exp(static_cast<double>(l[v]) - m);
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  unsigned long long key[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const double x = l[v];
    const double s = p.score == SB_SCORE_SOFTMAX ? exp(x - m) / sum : 1.0 / (1.0 + exp(-x));
    const double c = (l[v] == -INFINITY || b[v] == -INFINITY) ? -INFINITY : s + static_cast<double>(b[v]);
    key[v] = lane + 32 * v < p.E ? order_key(c) : 0;
  }
  bool unused = false;
  if (p.topk_groups < p.groups) keep_groups<V, false>(key, ch, p, lane, 0.f, &unused);
  return select_top<V, false>(key, l, b, p.K, lane, 0.f, &unused);
}

template <typename T, int V>
__global__ void __launch_bounds__(256) route_experts_kernel(const T* __restrict__ logits, const RouteParams p) {
  extern __shared__ __align__(16) uint8_t route_smem[];
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + warp;
  if (t >= p.n) return;
  unsigned long long* ch64 = reinterpret_cast<unsigned long long*>(route_smem) + static_cast<size_t>(warp) * p.E;
  float* s_sm = reinterpret_cast<float*>(ch64);
  const T* row = logits + t * p.ld;
  float l[V], b[V], s[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = lane + 32 * v;
    l[v] = e < p.E ? to_f32<T>(row[e]) : -INFINITY;
    b[v] = e < p.E && p.bias ? p.bias[e] : 0.f;
  }
  float sum = 0.f;
  if (p.score == SB_SCORE_SOFTMAX) {
    float m = -INFINITY;
#pragma unroll
    for (int v = 0; v < V; ++v) m = fmaxf(m, l[v]);
    m = warp_max(m);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      s[v] = l[v] == -INFINITY ? 0.f : expf(l[v] - m);
      sum += s[v];
    }
    sum = warp_sum(sum);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int v = 0; v < V; ++v) s[v] *= inv;
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) s[v] = 1.f / (1.f + expf(-l[v]));
  }
  const bool grouped = p.topk_groups < p.groups;
  const bool by_logit = !p.bias && !(grouped && p.group_top == 2);
  uint32_t key[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    // a NaN anywhere in a softmax row makes every score of the row NaN
    const float c = by_logit ? l[v] + 0.f * sum : ((l[v] == -INFINITY || b[v] == -INFINITY) ? -INFINITY : s[v] + b[v]);
    key[v] = lane + 32 * v < p.E ? order_key(c) : 0;
  }
  // fp32 error of a score: exp of a rounded difference (|x| e^-|x| 2^-24 <=
  // 0.37 2^-24), 2 ulp of expf, the sum and the division, all below 2^-20 in
  // all; two of them may differ by 2^-19.
  constexpr float kTol = 0x1p-19f;
  bool close = false;
  int mine;
  if (by_logit) {
    if (grouped) keep_groups<V, false>(key, reinterpret_cast<uint32_t*>(ch64), p, lane, 0.f, &close);
    mine = select_top<V, false>(key, l, b, p.K, lane, 0.f, &close);
  } else {
    if (grouped) keep_groups<V, true>(key, reinterpret_cast<uint32_t*>(ch64), p, lane, kTol, &close);
    mine = select_top<V, true>(key, l, b, p.K, lane, kTol, &close);
    if (close) mine = select_f64<V>(l, b, p, ch64, lane);
  }
  __syncwarp();
#pragma unroll
  for (int v = 0; v < V; ++v)
    if (lane + 32 * v < p.E) s_sm[lane + 32 * v] = (l[v] == -INFINITY || b[v] == -INFINITY) ? 0.f : s[v];
  __syncwarp();
  float w = lane < p.K ? s_sm[mine] : 0.f;
  if (p.renorm) {
    const float sum = warp_sum(w);
    w /= sum < 1e-9f ? 1e-9f : sum;  // not fmaxf, which would hide a NaN
  }
  if (lane < p.K) {
    p.top_idx[t * p.K + lane] = mine;
    p.top_w[t * p.K + lane] = w * p.scale;
  }
}

// Gradient of the weights with respect to the logits, the selection held fixed:
//   ds_j = scale (g_j - (sum_k g_k s_k) / D) / D   (renormalised, D = sum s)
//   ds_j = scale g_j / D'                          (D' = 1, or the floor 1e-9)
//   softmax: dl_i = s_i (ds_i - sum_k ds_k s_k);  sigmoid: dl_j = ds_j s_j (1 - s_j)
template <typename T, int V>
__global__ void __launch_bounds__(256)
route_experts_backward_kernel(const T* __restrict__ logits, const RouteParams p, const float* __restrict__ gw,
                              T* __restrict__ dl, int64_t ldd) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + warp;
  if (t >= p.n) return;
  const T* row = logits + t * p.ld;
  float l[V], s[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = lane + 32 * v;
    l[v] = e < p.E ? to_f32<T>(row[e]) : -INFINITY;
  }
  const int sel = lane < p.K ? p.top_idx[t * p.K + lane] : -1;
  const bool in_range = sel >= 0 && sel < p.E;
  const float g = in_range ? gw[t * p.K + lane] : 0.f;
  const float lsel = in_range ? to_f32<T>(row[sel]) : -INFINITY;
  const bool masked = lsel == -INFINITY || (p.bias && in_range && p.bias[sel] == -INFINITY);
  float ssel;
  if (p.score == SB_SCORE_SOFTMAX) {
    float m = -INFINITY;
#pragma unroll
    for (int v = 0; v < V; ++v) m = fmaxf(m, l[v]);
    m = warp_max(m);
    float sum = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      s[v] = l[v] == -INFINITY ? 0.f : expf(l[v] - m);
      sum += s[v];
    }
    sum = warp_sum(sum);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int v = 0; v < V; ++v) s[v] *= inv;
    ssel = lsel == -INFINITY ? 0.f : expf(lsel - m) * inv;
  } else {
    ssel = 1.f / (1.f + expf(-lsel));
  }
  const float sw = masked ? 0.f : ssel;  // the score that entered the weights
  float ds = p.scale * g;
  if (p.renorm) {
    const float sum = warp_sum(sw);
    const float d = sum < 1e-9f ? 1e-9f : sum;
    const float dot = warp_sum(g * sw);
    ds = p.scale * (sum < 1e-9f ? g : g - dot / d) / d;
  }
  if (masked) ds = 0.f;
  float add = ds * ssel * (1.f - ssel);  // sigmoid
  float dot = 0.f;
  if (p.score == SB_SCORE_SOFTMAX) {
    dot = warp_sum(ds * ssel);
    add = ds;
  }
  float dv[V];
#pragma unroll
  for (int v = 0; v < V; ++v) dv[v] = 0.f;
  for (int j = 0; j < p.K; ++j) {
    const int e = __shfl_sync(0xffffffffu, sel, j);
    const float a = __shfl_sync(0xffffffffu, add, j);
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (lane + 32 * v == e) dv[v] = a;
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = lane + 32 * v;
    if (e < p.E) dl[t * ldd + e] = from_f32<T>(p.score == SB_SCORE_SOFTMAX ? s[v] * (dv[v] - dot) : dv[v]);
  }
}

static bool route_args_ok(int dtype, int64_t ld, int n, int E, int K, int score) {
  return (dtype == SB_F32 || dtype == SB_BF16) && n >= 0 && E > 0 && E <= kRouteMaxE && K > 0 && K <= E &&
         K <= kRouteMaxK && ld >= E && (score == SB_SCORE_SOFTMAX || score == SB_SCORE_SIGMOID);
}

static int route_warps(int E) { return E <= 256 ? 8 : 4; }

template <typename T, int V>
static int launch_route(const void* logits, const RouteParams& p, cudaStream_t st) {
  const int warps = route_warps(p.E);
  const size_t smem = static_cast<size_t>(warps) * p.E * 8;  // at most 4 * 1024 * 8 = 32 KB
  return launch(route_experts_kernel<T, V>, dim3((p.n + warps - 1) / warps), dim3(warps * 32), smem, st,
                static_cast<const T*>(logits), p);
}

template <typename T, int V>
static int launch_route_backward(const void* logits, const RouteParams& p, const float* gw, void* dl, int64_t ldd,
                                 cudaStream_t st) {
  const int warps = route_warps(p.E);
  return launch(route_experts_backward_kernel<T, V>, dim3((p.n + warps - 1) / warps), dim3(warps * 32), 0, st,
                static_cast<const T*>(logits), p, gw, static_cast<T*>(dl), ldd);
}

#define SB_ROUTE_DISPATCH(FN, ...)                                              \
  do {                                                                          \
    const int v = (p.E + 31) / 32;                                              \
    if (dtype == SB_F32) {                                                      \
      if (v <= 1) return FN<float, 1>(__VA_ARGS__);                             \
      if (v <= 2) return FN<float, 2>(__VA_ARGS__);                             \
      if (v <= 4) return FN<float, 4>(__VA_ARGS__);                             \
      if (v <= 8) return FN<float, 8>(__VA_ARGS__);                             \
      if (v <= 16) return FN<float, 16>(__VA_ARGS__);                           \
      return FN<float, 32>(__VA_ARGS__);                                        \
    }                                                                           \
    if (v <= 1) return FN<__nv_bfloat16, 1>(__VA_ARGS__);                       \
    if (v <= 2) return FN<__nv_bfloat16, 2>(__VA_ARGS__);                       \
    if (v <= 4) return FN<__nv_bfloat16, 4>(__VA_ARGS__);                       \
    if (v <= 8) return FN<__nv_bfloat16, 8>(__VA_ARGS__);                       \
    if (v <= 16) return FN<__nv_bfloat16, 16>(__VA_ARGS__);                     \
    return FN<__nv_bfloat16, 32>(__VA_ARGS__);                                  \
  } while (0)

}  // namespace sb

using namespace sb;

extern "C" SB_API int sb_route_experts(const void* logits, int dtype, int64_t ld, int n_tokens, int num_experts,
                                       int top_k, int score, const float* bias, int num_groups, int topk_groups,
                                       int group_top, int renormalize, float scale, int32_t* top_idx, float* top_w,
                                       void* stream) {
  if (!route_args_ok(dtype, ld, n_tokens, num_experts, top_k, score) || num_groups < 1 ||
      num_groups > kRouteMaxGroups || num_experts % num_groups || topk_groups < 1 || topk_groups > num_groups ||
      top_k > topk_groups * (num_experts / num_groups) || (group_top != 1 && group_top != 2))
    return SB_ERR_ARG;
  if (n_tokens == 0) return SB_OK;
  if (!logits || !top_idx || !top_w) return SB_ERR_ARG;
  RouteParams p = {ld, n_tokens, num_experts, top_k, score, bias, num_groups, topk_groups, group_top, renormalize,
                   scale, top_idx, top_w};
  SB_ROUTE_DISPATCH(launch_route, logits, p, static_cast<cudaStream_t>(stream));
}

extern "C" SB_API int sb_route_experts_backward(const void* logits, int dtype, int64_t ld, int n_tokens,
                                                int num_experts, int top_k, int score, const float* bias,
                                                int renormalize, float scale, const int32_t* top_idx,
                                                const float* grad_w, void* grad_logits, int64_t ld_grad,
                                                void* stream) {
  if (!route_args_ok(dtype, ld, n_tokens, num_experts, top_k, score) || ld_grad < num_experts) return SB_ERR_ARG;
  if (n_tokens == 0) return SB_OK;
  if (!logits || !top_idx || !grad_w || !grad_logits) return SB_ERR_ARG;
  RouteParams p = {ld, n_tokens, num_experts, top_k, score, bias, 1, 1, 1, renormalize, scale,
                   const_cast<int32_t*>(top_idx), nullptr};
  SB_ROUTE_DISPATCH(launch_route_backward, logits, p, grad_w, grad_logits, ld_grad, static_cast<cudaStream_t>(stream));
}
