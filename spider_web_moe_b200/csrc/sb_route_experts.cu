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
// token with a gap inside the fp32 error is decided again, exactly: from fp64
// scores, or from the logits where the choices are monotonic in them (no bias).
//
// Bound by instructions, not memory: the fewest per token were found with the
// experts of a lane sorted once, and then one warp maximum per expert taken.
#include "sb_common.cuh"
#include "sb_internal.h"

namespace sb {

constexpr int kRouteMaxE = 1024;
constexpr int kRouteMaxK = 32;
constexpr int kRouteMaxGroups = 32;

// Order-preserving integer of a float: NaN above +inf, -0 equal to +0; every
// value, -inf too, is above 0, which marks an expert that is not a candidate.
SB_DEVINL uint32_t order_key(float v) {
  const uint32_t u = __float_as_uint(v + 0.0f);  // the sum of a NaN is the positive NaN
  return u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}
SB_DEVINL unsigned long long order_key(double v) {
  if (v != v) return ~0ull;
  const unsigned long long u = static_cast<unsigned long long>(__double_as_longlong(v + 0.0));
  return (u >> 63) ? ~u : (u | (1ull << 63));
}
SB_DEVINL float key_value(uint32_t k) {
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
  int per_group;    // E / groups
  int group_shift;  // a group is 2^group_shift whole lanes of the kernel's V experts, or -1
};

// Lane i holds the V experts [i V, i V + V): a lower lane means lower ids, so the
// lowest lane that holds the largest choice has the expert that wins a tie.

// A token's logits (-inf past E).  kVec: rows are aligned for whole-lane loads
// and E is a multiple of V.
template <typename T, int V, bool kVec>
SB_DEVINL void load_logits(const T* __restrict__ row, int E, int lane, float (&l)[V]) {
  const int e0 = lane * V;
  if constexpr (kVec) {
    constexpr int kBytes = V * sizeof(T);
    constexpr int kWords = kBytes / 4;
    uint32_t w[kWords];
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
    if (e0 < E) {
      if constexpr (kBytes >= 16) {
#pragma unroll
        for (int i = 0; i < kWords; i += 4) {
          const uint4 u = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(row + e0) + 4 * i);
          w[i] = u.x; w[i + 1] = u.y; w[i + 2] = u.z; w[i + 3] = u.w;
        }
      } else if constexpr (kBytes == 8) {
        const uint2 u = *reinterpret_cast<const uint2*>(row + e0);
        w[0] = u.x; w[1] = u.y;
      } else {
        w[0] = *reinterpret_cast<const uint32_t*>(row + e0);
      }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float x = sizeof(T) == 4 ? __uint_as_float(w[v])
                                     : __uint_as_float(v & 1 ? w[v / 2] & 0xffff0000u : w[v / 2] << 16);
      l[v] = e0 < E ? x : -INFINITY;
    }
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) l[v] = e0 + v < E ? to_f32<T>(row[e0 + v]) : -INFINITY;
  }
}

// The keys of the fast selection: the order key with its last bits replaced by
// the expert's place in the lane, so that a lane's experts sort with one minimum
// and one maximum per exchange, equal choices by lower id.  What the bits lose
// is below the closeness tolerance, or caught by it.
template <int V>
constexpr uint32_t kPlaceMask = V - 1;

SB_DEVINL float rcp_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// The choice of a key without the place: not below -inf, whose last bits it took.
SB_DEVINL float place_key_value(uint32_t k) { return key_value(max(k, 0x007fffffu)); }

template <int V>
SB_DEVINL void sort_descending(uint32_t (&k)[V]) {
#pragma unroll
  for (int size = 2; size <= V; size <<= 1)
#pragma unroll
    for (int d = size >> 1; d > 0; d >>= 1)
#pragma unroll
      for (int i = 0; i < V; ++i)
        if ((i & d) == 0) {
          const bool down = (i & size) == 0 || size == V;
          const uint32_t a = k[i], b = k[i | d];
          k[i] = down ? max(a, b) : min(a, b);
          k[i | d] = down ? min(a, b) : max(a, b);
        }
}

// The K largest of the lanes' sorted keys: lane j < K returns the j-th expert and
// its key without the place.  The lanes' lists lie in shared memory ([lane][V]);
// a lane holds the head of its list and moves on when it is taken.  *head: the
// head left at the end, *left how many keys lie before it.
template <int V>
SB_DEVINL int take_top(const uint32_t (&key)[V], uint32_t* list, uint32_t* taken, int K, int lane, uint32_t* mine_key,
                       uint32_t* head_out, int* used) {
  uint32_t* mylist = list + lane * V;
  if constexpr (V >= 4) {
#pragma unroll
    for (int v = 0; v < V; v += 4)
      *reinterpret_cast<uint4*>(mylist + v) = make_uint4(key[v], key[v + 1], key[v + 2], key[v + 3]);
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) mylist[v] = key[v];
  }
  uint32_t head = key[0];
  const uint32_t me = 1u << lane;
  const uint32_t last_id = static_cast<uint32_t>(lane * V) + kPlaceMask<V>;
  int at = 0;
  const uint32_t list_addr = smem_u32(mylist);
  const uint32_t taken_addr = smem_u32(taken);
  for (int j = 0; j < K; ++j) {
    const uint32_t h = head & ~kPlaceMask<V>;
    const uint32_t top = __reduce_max_sync(0xffffffffu, h);
    const uint32_t who = __ballot_sync(0xffffffffu, h == top);
    // the lowest lane of them writes its expert and moves on: predicated, so that
    // the round has no branch to reconverge from
    const uint32_t id = last_id - (head & kPlaceMask<V>);
    asm volatile(
        "{\n\t.reg .pred w, m;\n\t"
        "setp.eq.u32 w, %2, %3;\n\t"
        "@w st.shared.v2.b32 [%4], {%5, %6};\n\t"
        "@w add.s32 %0, %0, 1;\n\t"
        "setp.lt.and.s32 m, %0, %8, w;\n\t"
        "@w mov.b32 %1, 0;\n\t"
        "@m ld.shared.b32 %1, [%7];\n\t}"
        : "+r"(at), "+r"(head)
        : "r"(who & (0u - who)), "r"(me), "r"(taken_addr + 8 * j), "r"(id), "r"(h), "r"(list_addr + 4 * (at + 1)), "n"(V)
        : "memory");
  }
  __syncwarp();
  *head_out = head;
  *used = at;
  const uint2 t = lane < K ? *reinterpret_cast<const uint2*>(taken + 2 * lane) : make_uint2(0, 0);
  *mine_key = t.y;
  return static_cast<int>(t.x);
}

// The exact form: keys by place in the lane.  Lane j < K returns the j-th expert.
template <int V>
SB_DEVINL int take_top_exact(unsigned long long (&key)[V], int K, int lane) {
  int mine = 0;
  for (int j = 0; j < K; ++j) {
    unsigned long long best = key[0];
#pragma unroll
    for (int v = 1; v < V; ++v) best = key[v] > best ? key[v] : best;
    const unsigned long long top = warp_max_key(best);
    const int winner = __ffs(__ballot_sync(0xffffffffu, best == top)) - 1;
    int at = 0;  // the lowest expert of this lane that has the largest key
#pragma unroll
    for (int v = V - 1; v >= 0; --v)
      if (key[v] == top) at = v;
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (lane == winner && v == at) key[v] = 0;
    const int e = __shfl_sync(0xffffffffu, lane * V + at, winner);
    if (lane == j) mine = e;
  }
  return mine;
}

// Best two keys of each group, in lane g < groups.  k1 / k2: this lane's best
// two.  Groups of a power of two of whole lanes meet by shuffles; others scan the
// warp's keys in shared memory.
template <int V, typename Key>
SB_DEVINL void group_best(const Key (&key)[V], Key& k1, Key& k2, Key* ch, const RouteParams& p, int lane,
                          bool sorted) {
  if (p.group_shift >= 0) {
    const int lanes = 1 << p.group_shift;
    for (int o = 1; o < lanes; o <<= 1) {
      const Key o1 = __shfl_xor_sync(0xffffffffu, k1, o), o2 = __shfl_xor_sync(0xffffffffu, k2, o);
      const Key lo = o1 < k1 ? o1 : k1;
      k1 = o1 > k1 ? o1 : k1;
      k2 = o2 > k2 ? o2 : k2;
      k2 = lo > k2 ? lo : k2;
    }
    const int src = (lane << p.group_shift) & 31;
    k1 = __shfl_sync(0xffffffffu, k1, src);
    k2 = __shfl_sync(0xffffffffu, k2, src);
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int at = lane * V + (sorted ? static_cast<int>(kPlaceMask<V> - (key[v] & kPlaceMask<V>)) : v);
      if (key[v] != 0 && at < p.E) ch[at] = key[v];
    }
    __syncwarp();
    k1 = k2 = 0;
    for (int i = 0; lane < p.groups && i < p.per_group; ++i) {
      const Key k = ch[lane * p.per_group + i];
      if (k > k1) { k2 = k1; k1 = k; } else if (k > k2) k2 = k;
    }
    __syncwarp();
  }
}

// Bit mask of the best topk_groups groups, group g's score in lane g; *last is
// the key of the last one kept, gk afterwards 0 in the kept groups' lanes.
template <typename Key>
SB_DEVINL uint32_t best_groups(Key& gk, int topk_groups, int lane, Key* last) {
  uint32_t kept = 0;
  for (int j = 0; j < topk_groups; ++j) {
    *last = warp_max_key(gk);
    const int g = __ffs(__ballot_sync(0xffffffffu, gk == *last)) - 1;
    kept |= 1u << g;
    gk = lane == g ? 0 : gk;
  }
  return kept;
}

// The exact selection: from fp64 scores, or (by_logit) from the logits.  Rare, so
// it reads the logits again rather than have the caller keep them.
template <typename T, int V>
__device__ __noinline__ int select_exact(const T* __restrict__ row, const RouteParams& p, bool by_logit,
                                         unsigned long long* ch, int lane) {
  double m = 0.0, sum = 0.0;
  if (p.score == SB_SCORE_SOFTMAX && !by_logit) {
    float mf = -INFINITY;
    for (int v = 0; v < V; ++v)
      if (lane * V + v < p.E) mf = fmaxf(mf, to_f32<T>(row[lane * V + v]));
    m = warp_max(mf);
    for (int v = 0; v < V; ++v) {
      const float x = lane * V + v < p.E ? to_f32<T>(row[lane * V + v]) : -INFINITY;
      if (x != -INFINITY) sum += exp(static_cast<double>(x) - m);
    }
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  unsigned long long key[V], k1 = 0, k2 = 0;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = lane * V + v;
    key[v] = 0;
    if (e < p.E) {
      const float l = to_f32<T>(row[e]), b = p.bias ? p.bias[e] : 0.f;
      const double x = l;
      double c = x;
      if (!by_logit) {
        const double s = p.score == SB_SCORE_SOFTMAX ? exp(x - m) / sum : 1.0 / (1.0 + exp(-x));
        c = (l == -INFINITY || b == -INFINITY) ? -INFINITY : s + static_cast<double>(b);
      }
      key[v] = order_key(c);
    }
    const unsigned long long lo = key[v] < k1 ? key[v] : k1;
    k1 = key[v] > k1 ? key[v] : k1;
    k2 = lo > k2 ? lo : k2;
  }
  if (p.topk_groups < p.groups) {
    group_best<V>(key, k1, k2, ch, p, lane, false);
    double gs = key_value(k1);
    if (p.group_top == 2 && p.per_group > 1) gs += key_value(k2);
    unsigned long long gk = lane < p.groups ? order_key(gs) : 0, last;
    const uint32_t kept = best_groups(gk, p.topk_groups, lane, &last);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int e = lane * V + v;
      if (e < p.E && !((kept >> (e / p.per_group)) & 1u)) key[v] = 0;
    }
  }
  return take_top_exact<V>(key, p.K, lane);
}

// Shared memory per warp: the lanes' lists and the K experts taken, or (exact
// selection) fp64 keys of all experts.
template <int V>
constexpr int kRouteSmem = 32 * V * 8 + kRouteMaxK * 8;

template <typename T, int V, bool kVec>
__global__ void __launch_bounds__(256) route_experts_kernel(const T* __restrict__ logits,
                                                            const __grid_constant__ RouteParams p) {
  extern __shared__ __align__(16) uint8_t route_smem[];
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + warp;
  if (t >= p.n) return;
  unsigned long long* ch = reinterpret_cast<unsigned long long*>(route_smem + warp * kRouteSmem<V>);
  const T* row = logits + t * p.ld;
  const bool softmax = p.score == SB_SCORE_SOFTMAX;
  const bool grouped = p.topk_groups < p.groups;
  // without a bias the choices are monotonic in the logits, unless two are added
  const bool by_logit = !p.bias && !(grouped && p.group_top == 2);
  float l[V];
  load_logits<T, V, kVec>(row, p.E, lane, l);
  float m = -INFINITY, sum = 0.f, inv = 0.f, c[V];
  if (softmax) {
#pragma unroll
    for (int v = 0; v < V; ++v) m = fmaxf(m, l[v]);
    m = warp_max(m);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      c[v] = l[v] == -INFINITY ? 0.f : expf(l[v] - m);
      sum += c[v];
    }
    sum = warp_sum(sum);
    inv = sum == 0.f ? 0.f : 1.f / sum;
  }
  if (by_logit) {
    const float nan = 0.f * sum;  // a NaN anywhere in a softmax row makes every score of the row NaN
#pragma unroll
    for (int v = 0; v < V; ++v) c[v] = l[v] + nan;
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v)
      c[v] = softmax ? c[v] * inv : rcp_approx(1.f + __expf(-l[v]));
    if (p.bias) {
      float b[V];
      load_logits<float, V, kVec>(p.bias, p.E, lane, b);
#pragma unroll
      for (int v = 0; v < V; ++v) c[v] += b[v];
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) c[v] = l[v] == -INFINITY ? -INFINITY : c[v];
  uint32_t key[V];
#pragma unroll
  for (int v = 0; v < V; ++v)
    key[v] = lane * V + v < p.E ? (order_key(c[v]) & ~kPlaceMask<V>) | (kPlaceMask<V> - v) : 0;
  sort_descending<V>(key);
  // fp32 error of scores, in u = 2^-24.  Softmax, of s: V + 4 additions of the
  // sum, which can all round the same way, its terms (expf 4 u, and the rounded
  // differences x: their mean under the softmax weighs at most 5), expf again, the
  // division and the product: (V + 19) u s, and s |x| u <= 0.37 u for its own
  // difference.  The scores of two choices, or of the four of two group scores,
  // sum to at most 1: (V + 21) u between them.  Sigmoid: 4.6 u a score (the fast
  // exponential 2 + 1.17 |x| ulp times s (1 - s), the addition, the reciprocal),
  // 18.4 u for four.  Rounding of a choice: u of it, and V - 1 of its last places
  // for the expert's place.
  constexpr float kTol = (V + 24) * 0x1p-24f, kRel = (V + 1) * 0x1p-22f;
  // by_logit: the keys order exactly, but for the bits the place took (a bf16
  // logit has none there)
  const bool exact = by_logit && sizeof(T) == 2;
  bool close = false;
  if (grouped) {
    uint32_t k1 = key[0], k2 = V > 1 ? key[V > 1 ? 1 : 0] : 0;
    group_best<V>(key, k1, k2, reinterpret_cast<uint32_t*>(ch), p, lane, true);
    float gs = place_key_value(k1 & ~kPlaceMask<V>);
    if (p.group_top == 2 && p.per_group > 1) gs += place_key_value(k2 & ~kPlaceMask<V>);
    uint32_t gk = lane < p.groups ? order_key(gs) : 0, last;
    const uint32_t kept = best_groups(gk, p.topk_groups, lane, &last);
    if (by_logit) {
      close = !exact && gk != 0 && gk >= last;  // a group left out that is the equal of the last one kept
    } else {
      // The error of a sum goes by its terms, not by the sum: large ones of opposite
      // signs leave a small score known to little precision.  So the kept groups'
      // lower ends are compared with the upper ends of those left out.  (An infinite
      // score is exact: only infinite choices make it, or terms so large that no
      // finite score competes.)
      float err = 0.f;
      if (isfinite(gs)) {
        err = fabsf(place_key_value(k1 & ~kPlaceMask<V>));
        if (p.group_top == 2 && p.per_group > 1) err += fabsf(place_key_value(k2 & ~kPlaceMask<V>));
        err = 0.5f * kTol + 0.5f * kRel * err;
      }
      const bool group = lane < p.groups, in = group && ((kept >> lane) & 1u);
      const uint32_t low = ~warp_max_key(in ? ~order_key(gs - err) : 0u);  // the lowest of the kept
      close = group && !in && order_key(gs + err) >= low;
    }
    if (p.group_shift >= 0) {
      if (!((kept >> (lane >> p.group_shift)) & 1u)) {
#pragma unroll
        for (int v = 0; v < V; ++v) key[v] = 0;
      }
    } else {
      for (int v = 0; v < V; ++v) {
        const int e = lane * V + static_cast<int>(kPlaceMask<V> - (key[v] & kPlaceMask<V>));
        if (!((kept >> ((e / p.per_group) & 31)) & 1u)) key[v] = 0;
      }
      sort_descending<V>(key);  // the dropped ones to the end
    }
  }
  uint32_t mine_key, head;
  int used;
  uint32_t* list = reinterpret_cast<uint32_t*>(ch);
  int mine = take_top<V>(key, list, list + 32 * V, p.K, lane, &mine_key, &head, &used);
  float ls = lane < p.K ? to_f32<T>(row[mine]) : -INFINITY;
  float bs = lane < p.K && p.bias ? p.bias[mine] : 0.f;
  if (!exact) {
    // Did a decision hang on a gap that fp32 does not resolve?  Between one taken
    // expert and the next, or between the last taken and one left out, unless
    // the two are exactly equal (same logit, same bias).  (If such a gap lies
    // further up, the experts between are exactly equal to its upper end.)
    const uint32_t pk = __shfl_up_sync(0xffffffffu, mine_key, 1);
    const float pl = __shfl_up_sync(0xffffffffu, ls, 1), pb = __shfl_up_sync(0xffffffffu, bs, 1);
    const float cm = place_key_value(mine_key), pc = place_key_value(pk);
    const bool tight = by_logit ? pk == mine_key : pc - cm <= kTol + fabsf(pc) * kRel;
    close |= lane > 0 && lane < p.K && tight && (pl != ls || pb != bs);
    const uint32_t lk = __shfl_sync(0xffffffffu, mine_key, p.K - 1);
    const float lc = place_key_value(lk);
    const uint32_t limit = by_logit ? lk : order_key(lc - (kTol + fabsf(lc) * kRel));
    if (__any_sync(0xffffffffu, head >= limit)) {
      const float ll = __shfl_sync(0xffffffffu, ls, p.K - 1), lb = __shfl_sync(0xffffffffu, bs, p.K - 1);
      for (int v = used; v < V; ++v) {
        const uint32_t k = list[lane * V + v];
        if (k < limit || k == 0) break;
        const int e = lane * V + static_cast<int>(kPlaceMask<V> - (k & kPlaceMask<V>));
        close |= to_f32<T>(row[e]) != ll || (p.bias ? p.bias[e] : 0.f) != lb;
      }
      __syncwarp();
    }
    if (__any_sync(0xffffffffu, close)) {
      mine = select_exact<T, V>(row, p, by_logit && sum == sum, ch, lane);
      ls = lane < p.K ? to_f32<T>(row[mine]) : -INFINITY;
      bs = lane < p.K && p.bias ? p.bias[mine] : 0.f;
    }
  }
  float w = 0.f;
  if (lane < p.K && ls != -INFINITY && bs != -INFINITY)
    w = softmax ? expf(ls - m) * inv : 1.f / (1.f + expf(-ls));
  if (p.renorm) {
    const float total = warp_sum(w);
    w /= total < 1e-9f ? 1e-9f : total;  // not fmaxf, which would hide a NaN
  }
  if (lane < p.K) {
    p.top_idx[t * p.K + lane] = mine;
    p.top_w[t * p.K + lane] = w * p.scale;
  }
}

// Gradient of the weights with respect to the logits, the selection held fixed:
//   ds_j = scale (sum_k s_k (g_j - g_k) / D) / D   (renormalised, D = sum s)
//   ds_j = scale g_j / D'                          (D' = 1, or the floor 1e-9)
// The sum of differences does not cancel: it is exactly 0 where all g are equal,
// a single expert's among them.
//   softmax: dl_i = s_i (ds_i - sum_k ds_k s_k);  sigmoid: dl_j = ds_j s_j (1 - s_j)
template <typename T, int V, bool kVec>
__global__ void __launch_bounds__(256)
route_experts_backward_kernel(const T* __restrict__ logits, const __grid_constant__ RouteParams p, const float* __restrict__ gw,
                              T* __restrict__ dl, int64_t ldd) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + warp;
  if (t >= p.n) return;
  const T* row = logits + t * p.ld;
  const int sel = lane < p.K ? p.top_idx[t * p.K + lane] : -1;
  const bool in_range = sel >= 0 && sel < p.E;
  const float g = in_range ? gw[t * p.K + lane] : 0.f;
  const float lsel = in_range ? to_f32<T>(row[sel]) : -INFINITY;
  const bool masked = lsel == -INFINITY || (p.bias && in_range && p.bias[sel] == -INFINITY);
  float s[V];
  float ssel;
  if (p.score == SB_SCORE_SOFTMAX) {
    load_logits<T, V, kVec>(row, p.E, lane, s);
    float m = -INFINITY;
#pragma unroll
    for (int v = 0; v < V; ++v) m = fmaxf(m, s[v]);
    m = warp_max(m);
    float sum = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      s[v] = s[v] == -INFINITY ? 0.f : expf(s[v] - m);
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
    float diff = 0.f;
    for (int j = 0; j < p.K; ++j)
      diff = fmaf(__shfl_sync(0xffffffffu, sw, j), g - __shfl_sync(0xffffffffu, g, j), diff);
    ds = p.scale * (sum < 1e-9f ? g : diff / d) / d;
  }
  if (masked) ds = 0.f;
  float dv[V];
  float add;
  if (p.score == SB_SCORE_SOFTMAX) {
    // (renormalised, sum_k ds_k s_k is 0: only rounding would be left of it)
    const bool zero = p.renorm && warp_sum(sw) >= 1e-9f;
    const float dot = zero ? 0.f : warp_sum(ds * ssel);
#pragma unroll
    for (int v = 0; v < V; ++v) dv[v] = -dot;
    add = ds;
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      dv[v] = 0.f;
      s[v] = 1.f;
    }
    add = ds * ssel * (1.f - ssel);
  }
  for (int j = 0; j < p.K; ++j) {
    const int at = __shfl_sync(0xffffffffu, sel, j) - lane * V;
    const float a = __shfl_sync(0xffffffffu, add, j);
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (v == at) dv[v] += a;
  }
  T* out = dl + t * ldd + lane * V;
  if constexpr (kVec) {
    if (lane * V >= p.E) return;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int v = 0; v < V; v += 4)
        *reinterpret_cast<float4*>(out + v) =
            make_float4(s[v] * dv[v], s[v + 1] * dv[v + 1], s[v + 2] * dv[v + 2], s[v + 3] * dv[v + 3]);
    } else {
#pragma unroll
      for (int v = 0; v < V; v += 2)
        reinterpret_cast<__nv_bfloat162*>(out)[v / 2] = __floats2bfloat162_rn(s[v] * dv[v], s[v + 1] * dv[v + 1]);
    }
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (lane * V + v < p.E) out[v] = from_f32<T>(s[v] * dv[v]);
  }
}

static bool route_args_ok(int dtype, int64_t ld, int n, int E, int K, int score) {
  return (dtype == SB_F32 || dtype == SB_BF16) && n >= 0 && n <= kMaxExtent && E > 0 && E <= kRouteMaxE && K > 0 &&
         K <= E && K <= kRouteMaxK && ld >= E && (score == SB_SCORE_SOFTMAX || score == SB_SCORE_SIGMOID);
}

static int route_warps(int E) { return E <= 256 ? 8 : 4; }

// Whole-lane vector loads (and stores of the gradient): four or more experts a
// lane, all lanes full or empty, rows on 16-byte (or, below, on lane) boundaries.
template <typename T, int V>
static bool route_vec(const void* base, int64_t ld, int E) {
  constexpr int kBytes = V * sizeof(T) < 16 ? V * sizeof(T) : 16;
  return E % V == 0 && reinterpret_cast<uintptr_t>(base) % kBytes == 0 && ld * sizeof(T) % kBytes == 0;
}

template <typename T, int V>
static int launch_route(const void* logits, RouteParams p, cudaStream_t st) {
  const int warps = route_warps(p.E);
  const size_t smem = static_cast<size_t>(warps) * kRouteSmem<V>;  // at most 33 KB
  const int lanes = p.per_group / V;
  if (lanes * V == p.per_group && (lanes & (lanes - 1)) == 0) {
    p.group_shift = 0;
    while ((1 << p.group_shift) < lanes) ++p.group_shift;
  }
  const dim3 grid((p.n + warps - 1) / warps), block(warps * 32);
  if constexpr (V >= 4) {
    if (route_vec<T, V>(logits, p.ld, p.E) && (!p.bias || reinterpret_cast<uintptr_t>(p.bias) % 16 == 0))
      return launch(route_experts_kernel<T, V, true>, grid, block, smem, st, static_cast<const T*>(logits), p);
  }
  return launch(route_experts_kernel<T, V, false>, grid, block, smem, st, static_cast<const T*>(logits), p);
}

template <typename T, int V>
static int launch_route_backward(const void* logits, const RouteParams& p, const float* gw, void* dl, int64_t ldd,
                                 cudaStream_t st) {
  const int warps = route_warps(p.E);
  const dim3 grid((p.n + warps - 1) / warps), block(warps * 32);
  if constexpr (V >= 4) {
    if (route_vec<T, V>(logits, p.ld, p.E) && route_vec<T, V>(dl, ldd, p.E))
      return launch(route_experts_backward_kernel<T, V, true>, grid, block, 0, st, static_cast<const T*>(logits), p, gw,
                    static_cast<T*>(dl), ldd);
  }
  return launch(route_experts_backward_kernel<T, V, false>, grid, block, 0, st, static_cast<const T*>(logits), p, gw,
                static_cast<T*>(dl), ldd);
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
                   scale, top_idx, top_w, num_experts / num_groups, -1};
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
                   const_cast<int32_t*>(top_idx), nullptr, num_experts, -1};
  SB_ROUTE_DISPATCH(launch_route_backward, logits, p, grad_w, grad_logits, ld_grad, static_cast<cudaStream_t>(stream));
}
