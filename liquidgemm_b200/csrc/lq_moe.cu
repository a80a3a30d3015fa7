// Mixture-of-experts layer: the router, the plan that sorts (token, expert) pairs by expert, and what stands around the
// grouped products (lq_experts.cu): quantising the rows into their sorted places, the gated activation's quantiser and
// the weighted sum over a token's experts.
#include <cuda_runtime.h>

#include <mutex>

#include "lq_experts.cuh"
#include "lq_experts_epi.cuh"

namespace lq {
namespace experts {

// ---------------------------------------------------------------------------------------------
// router
// ---------------------------------------------------------------------------------------------
// One warp per token, expert e = lane + 32 i in register i of its lane.  Score s = softmax(l) over the token's experts or
// sigmoid(l).  Key: the logit itself without a bias (scores rise with it, and it is exact), else s + bias.  Groups of E / G
// neighbouring experts are ranked by their largest key or by the sum of their two largest keys (without a bias: scores), and
// only experts of the best groups stay.  Then `topk` times the largest key, the lowest index among equals.
// A logit of -inf or NaN, or a bias that makes a key so, takes its expert out.
//
// Where scores decide what is chosen (a bias, sums of two), neighbouring keys may lie closer than a float32 exponential's error, and
// a choice is a whole number.  The choice is made in float32 first; a token where two numbers whose order matters are closer than
// their errors together (about one in a thousand) is done again in float64.
//
// Bound by instruction issue and its latencies (a token's row is a few hundred bytes; with scores and groups 1390 instructions of a warp, the issue
// slots 65 % busy, the rest waits of a fixed length and for loads).  A choice is one 32-bit warp reduction, of 16-bit logits with the
// expert's index below them, or two, of the key and of the index; all lanes do the same throughout (the owner of a choice
// looking for its next best alone, and handing its score out by shuffles, took as long as all the rest).
// Groups are ranked from shared memory, 32 / G lanes to a group.  8192 tokens, 192 experts in 8 groups, sigmoid, bias: 64 us with
// a reduction of the 64-bit key for every group and choice, 22 with all of it in float64, 16 to 17 now.

// Orders numbers like unsigned integers; every number's image is above 0, which stands for "not to be chosen".
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t u = __float_as_uint(v + 0.0f);   // -0 becomes 0: equal keys are equal bits
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float number(uint32_t k) { return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu)); }
__device__ __forceinline__ unsigned long long ordered(double v) {
  const unsigned long long u = (unsigned long long)__double_as_longlong(v + 0.0);
  return u ^ ((u >> 63) ? 0xffffffffffffffffull : 0x8000000000000000ull);
}
__device__ __forceinline__ uint32_t warp_max(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }
__device__ __forceinline__ unsigned long long warp_max(unsigned long long v) {
  const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(v >> 32));
  const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(v >> 32) == hi ? (uint32_t)v : 0u);
  return ((unsigned long long)hi << 32) | lo;
}
template <typename S> struct KeyOf;
template <> struct KeyOf<float> { using type = uint32_t; };
template <> struct KeyOf<double> { using type = unsigned long long; };

// The upper 16 bits of a number that a 16-bit type holds, ordered like its 32-bit image.
template <typename T> __device__ __forceinline__ uint32_t ordered16(float v);
template <> __device__ __forceinline__ uint32_t ordered16<__nv_bfloat16>(float v) { return ordered(v) & 0xffff0000u; }
template <> __device__ __forceinline__ uint32_t ordered16<__half>(float v) {
  const uint32_t u = __half_as_ushort(__float2half_rn(v + 0.0f));   // exact: v came from a half
  return (u ^ ((u & 0x8000u) ? 0xffffu : 0x8000u)) << 16;
}
template <typename T> __device__ __forceinline__ float number16(uint32_t k);
template <> __device__ __forceinline__ float number16<__nv_bfloat16>(uint32_t k) {
  // (the image of a negative number has ones below, which its upper half lost)
  return number((k >> 31) ? (k & 0xffff0000u) : (k | 0xffffu));
}
template <> __device__ __forceinline__ float number16<__half>(uint32_t k) {
  const uint32_t u = k >> 16;
  return __half2float(__ushort_as_half((unsigned short)(u ^ ((u & 0x8000u) ? 0x8000u : 0xffffu))));
}

struct RouteArgs {
  const void* logits;
  const float* bias;
  float* weights;
  int* ids;
  int T, E, topk, n_group, topk_group;
  unsigned group_size, group_inv;   // E / n_group, and e / group_size = e * group_inv >> 20 for e < 512
  int group_lanes;                  // 32 / n_group down to a power of two, at least 1
  float scale;
  bool sigmoid, top2, renormalize;
};

constexpr int kRouteWarps = 4;
constexpr float kNone = -INFINITY;

// The logits of the warp's token; -inf for what cannot be chosen.
template <typename T, int PER>
__device__ __forceinline__ void load_logits(const RouteArgs& a, long t, float (&l)[PER]) {
  const T* row = static_cast<const T*>(a.logits) + t * a.E;
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = lane + 32 * i;
    l[i] = e < a.E ? to_f32<T>(row[e]) : kNone;
  }
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (!(l[i] > kNone)) l[i] = kNone;   // NaN too
}

// exp(l - top) of every expert (1 where equal: also where both are infinite) and their sum.
template <int PER, typename S>
__device__ __forceinline__ S softmax_terms(const float (&l)[PER], float& top, S (&s)[PER]) {
  top = kNone;
#pragma unroll
  for (int i = 0; i < PER; ++i) top = fmaxf(top, l[i]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  S sum = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    s[i] = !(l[i] > kNone) ? (S)0 : l[i] == top ? (S)1 : exp((S)l[i] - (S)top);
    sum += s[i];
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return sum > 0 ? sum : (S)1;
}

// Lane j has choice j (id -1: none left) and its logit l; softmax: `top` is the row's largest logit and `sum` the sum of exp(l - top) over all
// its experts (not used with renormalize).
//
// Renormalised softmax weights need the chosen logits alone: exp(l - m) over its sum, m the largest of the chosen.  A choice whose score (or,
// renormalised, weight) may lie near the end of float32's range, and only a row that has one, is worked out in float64: the ratio
// of such scores would be lost among float32's denormals.  What has no score in 64 bits (more than 745 below the top; a sigmoid below -709) has
// the weight 0.
__device__ __forceinline__ void store_choice(const RouteArgs& a, long t, int id, float l, float top, float sum) {
  const int lane = threadIdx.x & 31;
  const bool some = id >= 0;
  float ref = top;
  if (!a.sigmoid && a.renormalize) ref = number(__reduce_max_sync(0xffffffffu, some ? ordered(l) : 0u));
  const bool scored = some && (a.sigmoid || ref == top || ref - top > -745.f);
  float w = 0.f;
  if (__any_sync(0xffffffffu, some && (a.sigmoid ? l < -80.f : l - ref < -80.f))) {
    double s = 0.0;
    if (scored) s = a.sigmoid ? 1.0 / (1.0 + exp(-(double)l)) : l == ref ? 1.0 : exp((double)l - (double)ref);
    double total = 1.0;
    if (a.renormalize) {
      total = s;
      for (int o = 1; o < a.topk; o <<= 1) total += __shfl_xor_sync(0xffffffffu, total, o);   // (lanes behind the last slot hold 0)
      if (!(total > 0.0)) total = 1.0;
    } else if (!a.sigmoid) {
      total = sum;
    }
    w = (float)(s / total * a.scale);
  } else {
    if (scored) w = a.sigmoid ? __fdividef(1.f, 1.f + expf(-l)) : l == ref ? 1.f : expf(l - ref);
    float total = sum;
    if (a.renormalize) {
      total = w;
      for (int o = 1; o < a.topk; o <<= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    }
    if ((a.renormalize || !a.sigmoid) && total > 0.f) w = __fdiv_rn(w, total);
    w *= a.scale;
  }
  if (lane < a.topk) {
    a.weights[t * a.topk + lane] = w;
    a.ids[t * a.topk + lane] = id;
  }
}

// Which groups stay: those of the topk_group highest ranks, the lowest index among equals.  `v` [E]: what the groups are ranked by,
// -inf where an expert cannot be chosen; `rank` [n_group] and `kept` [n_group] are this warp's.  False where two ranks are closer than
// `near`.
template <typename S>
__device__ __forceinline__ bool rank_groups(const RouteArgs& a, bool top2, const S* v, S* rank, uint8_t* kept, S near) {
  const int lane = threadIdx.x & 31;
  const int G = a.n_group, size = (int)a.group_size, L = a.group_lanes, shift = __ffs(L) - 1;
  bool clear = true;
  for (int base = 0; base < G; base += 32 >> shift) {
    const int g = base + (lane >> shift);
    S m1 = kNone, m2 = kNone;
    if (g < G) {
      for (int e = lane & (L - 1); e < size; e += L) {
        const S x = v[g * size + e];
        m2 = x > m1 ? m1 : x > m2 ? x : m2;
        m1 = x > m1 ? x : m1;
      }
    }
    for (int o = 1; o < L; o *= 2) {
      const S b1 = __shfl_xor_sync(0xffffffffu, m1, o), b2 = __shfl_xor_sync(0xffffffffu, m2, o);
      const S least = m1 < b1 ? m1 : b1;
      m2 = m2 > b2 ? m2 : b2;
      m2 = least > m2 ? least : m2;
      m1 = m1 > b1 ? m1 : b1;
    }
    if (g < G && (lane & (L - 1)) == 0) {
      const bool two = top2 && m2 > (S)kNone;
      rank[g] = two ? m1 + m2 : m1;
      if (two && near >= 0 && fabs(m1 + m2) == (S)INFINITY) clear = false;   // a sum beyond float32, maybe
    }
  }
  __syncwarp();
  for (int g = lane; g < G; g += 32) {
    const S mine = rank[g];
    int before = 0;
    for (int o = 0; o < G; ++o) {
      const S other = rank[o];
      before += (other > mine || (other == mine && o < g)) ? 1 : 0;
      if (o != g && fabs(other - mine) <= near) clear = false;   // (-inf against -inf is NaN: clear)
    }
    kept[g] = before < a.topk_group;
  }
  __syncwarp();
  return __all_sync(0xffffffffu, clear);
}
__device__ __forceinline__ unsigned group_of(const RouteArgs& a, unsigned e) { return e * a.group_inv >> 20; }

// Choice by logits: no bias, groups by their largest.
template <typename T, int PER>
__global__ void __launch_bounds__(32 * kRouteWarps)
route_logits_kernel(const RouteArgs a) {
  __shared__ float values[kRouteWarps][PER * 32], ranks[kRouteWarps][PER * 32];
  __shared__ uint8_t kept[kRouteWarps][PER * 32];
  allow_dependents();
  dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long t = (long)blockIdx.x * kRouteWarps + warp;
  if (t >= a.T) return;
  constexpr bool k16 = sizeof(T) == 2;
  float l[PER];
  load_logits<T, PER>(a, t, l);
  uint32_t key[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = lane + 32 * i;
    if constexpr (k16) key[i] = l[i] > kNone ? ordered16<T>(l[i]) | (0xffffu - e) : 0u;
    else key[i] = l[i] > kNone ? ordered(l[i]) : 0u;
    if (a.n_group > 1) values[warp][e] = l[i];
  }
  if (a.n_group > 1) {
    __syncwarp();
    rank_groups<float>(a, false, values[warp], ranks[warp], kept[warp], -1.f);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const unsigned e = lane + 32 * i;
      if (e < a.E && !kept[warp][group_of(a, e)]) key[i] = 0;
    }
  }
  int my_id = -1;
  float my_l = 0.f;
  for (int j = 0; j < a.topk; ++j) {
    uint32_t mine = key[0];
#pragma unroll
    for (int i = 1; i < PER; ++i) mine = max(mine, key[i]);
    const uint32_t best = __reduce_max_sync(0xffffffffu, mine);
    if (best == 0) break;
    int id;
    if constexpr (k16) {
      id = (int)(0xffffu - (best & 0xffffu));
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (key[i] == best) key[i] = 0;
    } else {
      unsigned at = 1u << 20;
#pragma unroll
      for (int i = PER - 1; i >= 0; --i)
        if (key[i] == best) at = lane + 32 * i;
      id = (int)__reduce_min_sync(0xffffffffu, at);
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (id == lane + 32 * i) key[i] = 0;
    }
    if (lane == j) {
      my_id = id;
      if constexpr (k16) my_l = number16<T>(best);
      else my_l = number(best);
    }
  }
  float top = __shfl_sync(0xffffffffu, my_l, 0), sum = 1.f;   // the first choice is the row's largest logit: its group is the best
  if (!a.sigmoid && !a.renormalize) {
    float s[PER];
    sum = softmax_terms<PER, float>(l, top, s);
  }
  store_choice(a, t, my_id, my_l, top, sum);
}

// The warp's buffers of the kernel below.
template <int PER>
struct RouteBuffers {
  double values[PER * 32], ranks[PER * 32];
  uint8_t kept[PER * 32];
};

// Choice by scores.  False where the order of numbers that matters is not certain (float32 only).
// Errors of float32: a sigmoid is off by 6 * 2^-24 at most (exponential 2 units times e / (1 + e)^2, sum, quotient 2 units; 2^-21 is
// used), a softmax score by 31 * 2^-24 (argument |x| e^x < 0.4, exponential 2 units, sum of 16 terms and over 32 lanes, quotient;
// 2^-18 is used), the key by another |v| 2^-24; two keys by twice that, two sums of two by four times.
template <int PER, typename S>
__device__ __forceinline__ bool choose_by_score(const RouteArgs& a, const float (&l)[PER], RouteBuffers<PER>& buf, int& my_id, float& my_l,
                                                float& top, float& sum) {
  using Key = typename KeyOf<S>::type;
  constexpr bool kFast = sizeof(S) == 4;
  const int lane = threadIdx.x & 31;
  const bool by_score = a.bias != nullptr;
  S* values = reinterpret_cast<S*>(buf.values);
  S s[PER];
  if (a.sigmoid) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if constexpr (kFast) s[i] = l[i] > kNone ? __fdividef(1.f, 1.f + expf(-l[i])) : 0.f;
      else s[i] = l[i] > kNone ? 1.0 / (1.0 + exp(-(double)l[i])) : 0.0;
    }
  } else {
    const S all = softmax_terms<PER, S>(l, top, s);
    sum = (float)all;
#pragma unroll
    for (int i = 0; i < PER; ++i) s[i] = s[i] / all;
  }
  Key key[PER];
  S largest = 1;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = lane + 32 * i;
    S v = (S)kNone;
    if (l[i] > kNone) v = by_score ? s[i] + (S)a.bias[e] : (S)l[i];
    const bool can = v > (S)kNone;   // (false for NaN)
    key[i] = can ? ordered(v) : 0;
    if (kFast && by_score && can) largest = fabs(v) > largest ? fabs(v) : largest;
    if (a.n_group > 1) values[e] = !can ? (S)kNone : a.top2 && !by_score ? s[i] : v;
  }
  S near = (S)-1;
  if (kFast) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const S other = __shfl_xor_sync(0xffffffffu, largest, o);
      largest = other > largest ? other : largest;
    }
    near = (S)2 * ((a.sigmoid ? (S)0x1p-21f : (S)0x1p-18f) + largest * (S)0x1p-24f);
  }
  if (a.n_group > 1) {
    __syncwarp();
    const bool ranked_by_score = by_score || a.top2;
    if (!rank_groups<S>(a, a.top2, values, reinterpret_cast<S*>(buf.ranks), buf.kept, ranked_by_score ? (S)2 * near : (S)-1)) return false;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const unsigned e = lane + 32 * i;
      if (e < a.E && !buf.kept[group_of(a, e)]) key[i] = 0;
    }
  }
  // the chosen ones' weights are worked out from their logits, a lane each
  __syncwarp();
#pragma unroll
  for (int i = 0; i < PER; ++i) values[lane + 32 * i] = (S)l[i];
  __syncwarp();
  uint32_t last = 0;   // the choice before
  const bool check = kFast && by_score;
  for (int j = 0; j < a.topk + (check ? 1 : 0); ++j) {   // the first that is not chosen is looked at too
    Key mine = key[0];
#pragma unroll
    for (int i = 1; i < PER; ++i) mine = key[i] > mine ? key[i] : mine;
    const Key best = warp_max(mine);
    if (best == 0) break;
    if constexpr (kFast) {
      if (check && j > 0 && number(last) - number(best) <= near) return false;
      last = best;
    }
    if (j == a.topk) break;
    unsigned at = 1u << 20;
#pragma unroll
    for (int i = PER - 1; i >= 0; --i)
      if (key[i] == best) at = lane + 32 * i;
    const int id = (int)__reduce_min_sync(0xffffffffu, at);
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (id == lane + 32 * i) key[i] = 0;
    if (lane == j) my_id = id;
  }
  if (my_id >= 0) my_l = (float)values[my_id];
  return true;
}

template <typename T, int PER>
__global__ void __launch_bounds__(32 * kRouteWarps)
route_scores_kernel(const RouteArgs a) {
  __shared__ RouteBuffers<PER> buffers[kRouteWarps];
  allow_dependents();
  dependency_wait();
  const int warp = threadIdx.x >> 5;
  const long t = (long)blockIdx.x * kRouteWarps + warp;
  if (t >= a.T) return;
  float l[PER];
  load_logits<T, PER>(a, t, l);
  int id = -1;
  float my_l = 0.f, top = 0.f, sum = 1.f;
  if (!choose_by_score<PER, float>(a, l, buffers[warp], id, my_l, top, sum)) {
    __syncwarp();
    id = -1;
    choose_by_score<PER, double>(a, l, buffers[warp], id, my_l, top, sum);
  }
  store_choice(a, t, id, my_l, top, sum);
}

template <typename T, int PER>
static cudaError_t launch_route_per(const RouteArgs& a, cudaStream_t st) {
  const bool scores = a.bias != nullptr || (a.n_group > 1 && a.top2);
  return launch_overlapped(scores ? route_scores_kernel<T, PER> : route_logits_kernel<T, PER>,
                           dim3((a.T + kRouteWarps - 1) / kRouteWarps), dim3(32 * kRouteWarps), 0, st, a);
}
template <typename T>
static int launch_route(const RouteArgs& a, cudaStream_t st) {
  const int per = (a.E + 31) / 32;
  const cudaError_t e = per <= 1    ? launch_route_per<T, 1>(a, st)
                        : per <= 2  ? launch_route_per<T, 2>(a, st)
                        : per <= 4  ? launch_route_per<T, 4>(a, st)
                        : per <= 6  ? launch_route_per<T, 6>(a, st)
                        : per <= 8  ? launch_route_per<T, 8>(a, st)
                        : per <= 12 ? launch_route_per<T, 12>(a, st)
                                    : launch_route_per<T, 16>(a, st);
  if (e != cudaSuccess) {
    record_cuda_error(e, "route kernel launch");
    return LQ_ERR_CUDA;
  }
  return check_launch("route kernel");
}

// ---------------------------------------------------------------------------------------------
// plan
// ---------------------------------------------------------------------------------------------
// The tiles of expert e: as few as cover its n rows, and of equal widths in steps of 32 (a full tile and a narrow rest would
// take as long as two full ones wherever the two run side by side).  Every one has a row: bn is a multiple of 32.
// One warp; tiles and rows are lane 31's.  Each lane takes a number of ranges, the fewest of the best are kept.
__device__ __forceinline__ void write_counts(const Plan& plan, int tiles, int rows) {
  const int lane = threadIdx.x & 31;
  tiles = __shfl_sync(0xffffffffu, tiles, 31);
  int cuts[2];
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    cuts[w] = 1;
    if (plan.rule[w].most > 1) {
      const unsigned cost = lane < plan.rule[w].most ? split_cost(tiles, plan.rule[w], lane + 1, plan.slots) : 0xffffffffu;
      cuts[w] = __ffs(__ballot_sync(0xffffffffu, cost == __reduce_min_sync(0xffffffffu, cost)));
    } else if (plan.rule[w].even && cut_evenly(tiles, plan.rule[w], plan.slots)) {
      cuts[w] = 0;
    }
  }
  if (lane == 31) *reinterpret_cast<int4*>(plan.counts) = make_int4(tiles, rows, cuts[0], cuts[1]);
}
__device__ __forceinline__ void clear_joins(const Plan& plan, int thread, int threads) {
  for (int w = 0; w < 2; ++w)
    if (plan.rule[w].even)
      for (int i = thread; i < plan.slots; i += threads) plan.join[w][i] = make_int4(0, 0, 0, 0);
}
__device__ __forceinline__ void write_tiles(const Plan& plan, int tile0, int e, int row0, int n, int tiles) {
  if (tiles == 0) return;
  const int per = ((n + tiles - 1) / tiles + 31) & ~31;
  for (int i = 0; i < tiles; ++i) {
    const int left = n - i * per;
    plan.tiles[tile0 + i] = make_int4(e, row0 + i * per, left < per ? left : per, 0);
  }
}

// One CTA of 32 warps.  Warp w counts the pairs of its contiguous share per expert, the counts are summed over warps and
// experts, and in a second pass every pair's row is the running count of its (warp, expert): a stable sort, the same
// on every run.  Bound by the latency of its two passes over the ids (13332 pairs of 32 experts: 14 us).
constexpr int kPlanWarps = 32;
// The lanes whose number is this lane's, bit by bit; the numbers differ in the low `bits` bits only.  __match_any_sync takes the longer the
// more different numbers there are: the kernel takes 12.0 us with it and 13.2 with this for 16384 pairs of 8 experts, 16.0 and 13.8 for
// 13332 of 32, 84 and 59 for 65536 of 256.
__device__ __forceinline__ unsigned lanes_alike(int v, int bits) {
  unsigned same = 0xffffffffu;
  for (int b = 0; b < bits; ++b) {
    const bool one = (v >> b) & 1;
    const unsigned ones = __ballot_sync(0xffffffffu, one);
    same &= one ? ones : ~ones;
  }
  return same;
}
__global__ void __launch_bounds__(32 * kPlanWarps)
plan_kernel(const int* ids, long pairs, int E, const Plan plan) {
  extern __shared__ int hist[];   // [kPlanWarps][E]
  __shared__ int sums[2][kPlanWarps];
  allow_dependents();
  dependency_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < kPlanWarps * E; i += blockDim.x) hist[i] = 0;
  clear_joins(plan, threadIdx.x, blockDim.x);
  __syncthreads();
  const long share = ((pairs + kPlanWarps - 1) / kPlanWarps + 31) / 32 * 32;
  const long begin = warp * share, end = begin + share < pairs ? begin + share : pairs;
  constexpr int kAhead = 8;   // ids of a lane in flight
  for (long i0 = begin; i0 < end; i0 += 32 * kAhead) {
    int e[kAhead];
#pragma unroll
    for (int q = 0; q < kAhead; ++q) e[q] = i0 + 32 * q + lane < end ? ids[i0 + 32 * q + lane] : -1;
#pragma unroll
    for (int q = 0; q < kAhead; ++q)
      if (e[q] >= 0 && e[q] < E) atomicAdd(&hist[warp * E + e[q]], 1);
  }
  __syncthreads();
  // thread e: the pairs of expert e, and how many of them lie before each warp's share
  const int e = threadIdx.x;
  int n = 0, tiles = 0;
  int share_of[kPlanWarps];
  if (e < E) {
#pragma unroll
    for (int w = 0; w < kPlanWarps; ++w) share_of[w] = hist[w * E + e];
#pragma unroll
    for (int w = 0; w < kPlanWarps; ++w) {
      const int c = share_of[w];
      share_of[w] = n;
      n += c;
    }
    tiles = (n + plan.bn - 1) / plan.bn;
  }
  // exclusive sums over the experts of both counts
  int a = n, b = tiles;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int pa = __shfl_up_sync(0xffffffffu, a, o), pb = __shfl_up_sync(0xffffffffu, b, o);
    if (lane >= o) a += pa, b += pb;
  }
  if (lane == 31) sums[0][warp] = a, sums[1][warp] = b;
  __syncthreads();
  int ra = 0, rb = 0;
  for (int w = 0; w < warp; ++w) ra += sums[0][w], rb += sums[1][w];
  const int row0 = ra + a - n, tile0 = rb + b - tiles;
  if (e < E) {
#pragma unroll
    for (int w = 0; w < kPlanWarps; ++w) hist[w * E + e] = share_of[w] + row0;
    write_tiles(plan, tile0, e, row0, n, tiles);
  }
  if (warp == kPlanWarps - 1) write_counts(plan, rb + b, ra + a);
  __syncthreads();
  const int bits = 32 - __clz(E);   // of an expert's number, or of -1 beside them
  for (long i0 = begin; i0 < end; i0 += 32 * kAhead) {
    int id[kAhead];
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {
      id[q] = i0 + 32 * q + lane < end ? ids[i0 + 32 * q + lane] : -1;
      if (id[q] < 0 || id[q] >= E) id[q] = -1;
    }
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {
      if (i0 + 32 * q >= end) break;
      const long i = i0 + 32 * q + lane;
      const unsigned same = E < 16 ? __match_any_sync(0xffffffffu, id[q]) : lanes_alike(id[q], bits);
      const int before = __popc(same & ((1u << lane) - 1u));
      int base = 0;
      if (id[q] >= 0) base = hist[warp * E + id[q]];
      __syncwarp();
      if (id[q] >= 0 && before == 0) hist[warp * E + id[q]] = base + __popc(same);
      __syncwarp();
      if (i < end) {
        plan.pos_of_pair[i] = id[q] >= 0 ? base + before : -1;
        if (id[q] >= 0) plan.pair_of_pos[base + before] = (int)i;
      }
    }
  }
}

static int run_plan(const int* ids, long pairs, int E, const Plan& plan, cudaStream_t st) {
  const size_t smem = (size_t)kPlanWarps * E * sizeof(int);
  static std::once_flag once[64];
  int dev = 0;
  cudaGetDevice(&dev);
  std::call_once(once[dev & 63], [&]() {
    cudaFuncSetAttribute(plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kPlanWarps * kMaxExperts * (int)sizeof(int));
  });
  const cudaError_t e = launch_overlapped(plan_kernel, dim3(1), dim3(32 * kPlanWarps), smem, st, ids, pairs, E, plan);
  if (e != cudaSuccess) {
    record_cuda_error(e, "plan_kernel launch");
    return LQ_ERR_CUDA;
  }
  return check_launch("plan_kernel");
}

// ---------------------------------------------------------------------------------------------
// rows into their sorted places
// ---------------------------------------------------------------------------------------------
// One CTA per row of x (one per token, or one per pair): quantised as by quant_row_kernel of the dense linear, bit for bit,
// and written to the places of its pairs.  NV 16-byte vectors per thread in registers; NV = 0: a row too long for that is read
// twice.  Where the outputs are one row per pair, the rows of pairs without an expert are set to zero here.
//
// Up to kSortedHere pairs (SORT) there is no plan kernel before this one: a CTA finds the places of its own pairs
// by counting the pairs that come before them, and one more CTA (the first) cuts the experts' rows into tiles.  That
// saves a launch and its hand-over, 4 of the 9 us before the first product of a decode step; the counting grows with
// the square of the pairs (at 2048 it takes the time of the plan kernel).  A latency with few rows (one row of 4096: 3-5 us with its
// launch), bound by memory with many (13332 places of 3333 rows of 4096: 16 us).
constexpr int kSortedHere = 2048;
struct PlaceArgs {
  const void* x;
  const float* x_scale;    // scales of INT8 rows
  int8_t* xq;
  float* ascale;
  const int* pos_of_pair;
  unsigned* amax;          // set to zero for the rows placed, or null
  void* y;                 // [pairs, N] whose rows without an expert are cleared, or null
  int y_size;              // bytes of an element of y
  int per_row;             // pairs of a row of x
  int K, N;
  const int* ids;          // SORT: the pairs and where the plan goes
  int pairs, E;
  Plan plan;
};

// The ids into shared memory, once per CTA: every CTA wants all of them at the same time, and asked for by each of its warps they
// queue at the few L2 lines that hold them (1800 pairs: 8 us).
__device__ __forceinline__ void fetch_ids(const PlaceArgs& a, int* ids) {
  constexpr int kAhead = 8;   // of a thread in flight
  for (int i0 = threadIdx.x; i0 < a.pairs; i0 += kAhead * blockDim.x) {
    int e[kAhead];
#pragma unroll
    for (int q = 0; q < kAhead; ++q) e[q] = i0 + q * (int)blockDim.x < a.pairs ? a.ids[i0 + q * blockDim.x] : 0;
#pragma unroll
    for (int q = 0; q < kAhead; ++q)
      if (i0 + q * (int)blockDim.x < a.pairs) ids[i0 + q * blockDim.x] = e[q];
  }
}

// Tiles and counts of the plan (one CTA, of a single warp where the rows are short).
__device__ __forceinline__ void make_tiles(const PlaceArgs& a, int* hist) {
  clear_joins(a.plan, threadIdx.x, blockDim.x);
  for (int e = threadIdx.x; e < kMaxExperts; e += blockDim.x) hist[e] = 0;
  __syncthreads();
  constexpr int kAhead = 8;   // ids of a thread in flight
  for (int i0 = threadIdx.x; i0 < a.pairs; i0 += kAhead * blockDim.x) {
    int e[kAhead];
#pragma unroll
    for (int q = 0; q < kAhead; ++q) e[q] = i0 + q * (int)blockDim.x < a.pairs ? a.ids[i0 + q * blockDim.x] : -1;
#pragma unroll
    for (int q = 0; q < kAhead; ++q)
      if (e[q] >= 0 && e[q] < a.E) atomicAdd(&hist[e[q]], 1);
  }
  __syncthreads();
  if (threadIdx.x >= 32) return;
  const int per = (a.E + 31) / 32;   // neighbouring experts of a lane
  const int lane = threadIdx.x;
  int rows = 0, tiles = 0;
  for (int q = 0; q < per; ++q) {
    const int n = hist[lane * per + q];
    rows += n;
    tiles += (n + a.plan.bn - 1) / a.plan.bn;
  }
  int r = rows, t = tiles;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int pr = __shfl_up_sync(0xffffffffu, r, o), pt = __shfl_up_sync(0xffffffffu, t, o);
    if (lane >= o) r += pr, t += pt;
  }
  write_counts(a.plan, t, r);
  r -= rows;
  t -= tiles;
  for (int q = 0; q < per; ++q) {
    const int e = lane * per + q, n = hist[e];
    const int mine = (n + a.plan.bn - 1) / a.plan.bn;
    write_tiles(a.plan, t, e, r, n, mine);
    t += mine;
    r += n;
  }
}

// The places of the pairs of row m, in `place` [per_row] (shared memory): read from the plan, or counted (`ids`: room for all) and
// entered there.
template <bool SORT>
__device__ __forceinline__ void find_places(const PlaceArgs& a, long m, int* ids, int* place) {
  if constexpr (!SORT) {
    for (int j = threadIdx.x; j < a.per_row; j += blockDim.x) place[j] = a.pos_of_pair[m * a.per_row + j];
  } else {
    fetch_ids(a, ids);
    __syncthreads();
    const int lane = threadIdx.x & 31;
    for (int j = threadIdx.x >> 5; j < a.per_row; j += blockDim.x >> 5) {
      const int pair = (int)m * a.per_row + j;
      const int e = ids[pair];
      int before = 0;
#pragma unroll 8
      for (int i = lane; i < a.pairs; i += 32) {
        const int o = ids[i];
        before += (o >= 0 && (o < e || (o == e && i < pair))) ? 1 : 0;
      }
      before = __reduce_add_sync(0xffffffffu, before);
      if (lane == 0) {
        const bool some = e >= 0 && e < a.E;
        place[j] = some ? before : -1;
        a.plan.pos_of_pair[pair] = some ? before : -1;
        if (some) a.plan.pair_of_pos[before] = pair;
      }
    }
  }
}

__device__ __forceinline__ void clear_output_row(const PlaceArgs& a, long pair) {
  if (a.y_size == 2) {
    uint16_t* y = static_cast<uint16_t*>(a.y) + pair * a.N;
    for (int n = threadIdx.x; n < a.N; n += blockDim.x) y[n] = 0;
  } else {
    uint32_t* y = static_cast<uint32_t*>(a.y) + pair * a.N;
    for (int n = threadIdx.x; n < a.N; n += blockDim.x) y[n] = 0;
  }
}

template <typename T, int NV, bool SORT>
__global__ void __launch_bounds__(1024)
place_rows_kernel(const PlaceArgs a) {
  __shared__ float red[32];
  __shared__ int place[kMaxTopk];
  __shared__ int ids[SORT ? kSortedHere : 1];
  constexpr int VEC = 16 / sizeof(T);
  allow_dependents();
  dependency_wait();
  if (SORT && blockIdx.x == 0) {
    make_tiles(a, ids);
    return;
  }
  const long m = SORT ? blockIdx.x - 1 : blockIdx.x;
  const uint4* xr = reinterpret_cast<const uint4*>(static_cast<const T*>(a.x) + m * a.K);
  const int nvec = a.K / VEC;
  uint4 raw[NV > 0 ? NV : 1];
  RowMax<T> rm;
  if constexpr (NV > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = threadIdx.x + i * blockDim.x;
      raw[i] = v < nvec ? xr[v] : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) rm.take(raw[i]);
  } else {
    for (int v = threadIdx.x; v < nvec; v += blockDim.x) rm.take(xr[v]);
  }
  find_places<SORT>(a, m, ids, place);
  const float amax = block_max(rm.value(), red);   // (its barrier orders the places too)
  const float scale = __fdiv_rn(fmaxf(amax, 1e-12f), 127.0f);
  const float inv = __fdiv_rn(1.0f, scale);
  constexpr int kWords = 4 / sizeof(T);   // of four codes, from one vector
  uint32_t q[NV > 0 ? NV : 1][kWords];
  if constexpr (NV > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) quant_vec<T>(raw[i], scale, inv, q[i]);
  }
  for (int j = 0; j < a.per_row; ++j) {
    const long pair = m * a.per_row + j;
    const int p = place[j];
    if (p < 0) {
      if (a.y) clear_output_row(a, pair);
      continue;
    }
    if (threadIdx.x == 0) {
      a.ascale[p] = scale;
      if (a.amax) a.amax[p] = 0u;
    }
    uint32_t* qr = reinterpret_cast<uint32_t*>(a.xq + (long)p * a.K);
    if constexpr (NV > 0) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = threadIdx.x + i * blockDim.x;
        if (v >= nvec) break;
        if constexpr (kWords == 1) qr[v] = q[i][0];
        else reinterpret_cast<uint2*>(qr)[v] = make_uint2(q[i][0], q[i][1]);
      }
    } else {
      for (int v = threadIdx.x; v < nvec; v += blockDim.x) {
        quant_vec<T>(xr[v], scale, inv, q[0]);
        if constexpr (kWords == 1) qr[v] = q[0][0];
        else reinterpret_cast<uint2*>(qr)[v] = make_uint2(q[0][0], q[0][1]);
      }
    }
  }
}

// Rows that come in INT8 with their scales.
template <bool SORT>
__global__ void __launch_bounds__(256)
place_i8_kernel(const PlaceArgs a) {
  __shared__ int place[kMaxTopk];
  __shared__ int ids[SORT ? kSortedHere : 1];
  allow_dependents();
  dependency_wait();
  if (SORT && blockIdx.x == 0) {
    make_tiles(a, ids);
    return;
  }
  const long m = SORT ? blockIdx.x - 1 : blockIdx.x;
  find_places<SORT>(a, m, ids, place);
  __syncthreads();
  const uint4* xr = reinterpret_cast<const uint4*>(static_cast<const int8_t*>(a.x) + m * a.K);
  const float scale = a.x_scale[m];
  for (int j = 0; j < a.per_row; ++j) {
    const long pair = m * a.per_row + j;
    const int p = place[j];
    if (p < 0) {
      if (a.y) clear_output_row(a, pair);
      continue;
    }
    if (threadIdx.x == 0) a.ascale[p] = scale;
    uint4* qr = reinterpret_cast<uint4*>(a.xq + (long)p * a.K);
    for (int v = threadIdx.x; v < a.K / 16; v += blockDim.x) qr[v] = xr[v];
  }
}

template <typename T, bool SORT>
static cudaError_t launch_place(const PlaceArgs& a, long rows, cudaStream_t st) {
  int threads = 0;
  const int nv = row_units_per_thread(rows, a.K / (16 / (int)sizeof(T)), 8, 128, 1024, &threads);
  void (*kern)(PlaceArgs) = nv == 1   ? place_rows_kernel<T, 1, SORT>
                            : nv == 2 ? place_rows_kernel<T, 2, SORT>
                            : nv == 4 ? place_rows_kernel<T, 4, SORT>
                            : nv == 8 ? place_rows_kernel<T, 8, SORT>
                                      : place_rows_kernel<T, 0, SORT>;
  if (nv == 0) threads = 1024;
  return launch_overlapped(kern, dim3((unsigned)rows + (SORT ? 1u : 0u)), dim3(threads), 0, st, a);
}
template <bool SORT>
static int launch_place_any(const PlaceArgs& a, int x_dtype, long rows, cudaStream_t st) {
  const cudaError_t e = x_dtype == LQ_DT_BF16  ? launch_place<__nv_bfloat16, SORT>(a, rows, st)
                        : x_dtype == LQ_DT_F16 ? launch_place<__half, SORT>(a, rows, st)
                        : x_dtype == LQ_DT_F32 ? launch_place<float, SORT>(a, rows, st)
                                               : launch_overlapped(place_i8_kernel<SORT>, dim3((unsigned)rows + (SORT ? 1u : 0u)),
                                                                   dim3(256), 0, st, a);
  if (e != cudaSuccess) {
    record_cuda_error(e, "place kernel launch");
    return LQ_ERR_CUDA;
  }
  return check_launch("place kernel");
}

// Plan and rows.
static int run_place(PlaceArgs& a, const int* ids, long pairs, int E, const Plan& plan, int x_dtype, long rows, cudaStream_t st) {
  a.pos_of_pair = plan.pos_of_pair;
  if (pairs <= kSortedHere) {
    a.ids = ids;
    a.pairs = (int)pairs;
    a.E = E;
    a.plan = plan;
    return launch_place_any<true>(a, x_dtype, rows, st);
  }
  if (int rc = run_plan(ids, pairs, E, plan, st)) return rc;
  return launch_place_any<false>(a, x_dtype, rows, st);
}

// ---------------------------------------------------------------------------------------------
// hidden rows: activation (where the product left its sums) and quantisation
// ---------------------------------------------------------------------------------------------
struct HiddenArgs {
  const int32_t* planes;     // [splits][rows][2 * I] sums of the gate and up channels, interleaved; or null
  const float* h;            // [rows][I] hidden values, with amax
  const unsigned* amax;
  const float* ascale;       // [rows] scales of the product's rows
  const float* s1;           // [E][2 * I]
  const int* ids;            // [pairs]
  const int* counts;
  const int* pair_of_pos;
  int8_t* hq;                // [rows][I]
  float* hscale;             // [rows]
  long rows;
  int I;
};

// Four hidden values of row p from the planes.
__device__ __forceinline__ void hidden4(const HiddenArgs& a, int splits, long p, const float* s1, float as, int c, float (&h)[4]) {
  int4 g0 = make_int4(0, 0, 0, 0), g1 = g0;
  for (int s = 0; s < splits; ++s) {
    const int4* src = reinterpret_cast<const int4*>(a.planes + ((size_t)s * a.rows + p) * 2 * a.I + 2 * c);
    const int4 v0 = src[0], v1 = src[1];
    g0.x += v0.x; g0.y += v0.y; g0.z += v0.z; g0.w += v0.w;
    g1.x += v1.x; g1.y += v1.y; g1.z += v1.z; g1.w += v1.w;
  }
  const float4 f0 = *reinterpret_cast<const float4*>(s1 + 2 * c), f1 = *reinterpret_cast<const float4*>(s1 + 2 * c + 4);
  h[0] = gated(lqq_scale(g0.x, as, f0.x), lqq_scale(g0.y, as, f0.y));
  h[1] = gated(lqq_scale(g0.z, as, f0.z), lqq_scale(g0.w, as, f0.w));
  h[2] = gated(lqq_scale(g1.x, as, f1.x), lqq_scale(g1.y, as, f1.y));
  h[3] = gated(lqq_scale(g1.z, as, f1.z), lqq_scale(g1.w, as, f1.w));
}

__device__ __forceinline__ uint32_t quant4(const float (&h)[4], float scale, float inv) {
  uint32_t out[1];
  quant_vec<float>(make_uint4(__float_as_uint(h[0]), __float_as_uint(h[1]), __float_as_uint(h[2]), __float_as_uint(h[3])), scale,
                   inv, out);
  return out[0];
}

// One CTA per row: the largest magnitude first, then the codes; the row's values are worked out twice, from sums that the
// second pass finds in L2.  A latency: k is cut where rows are few.
__global__ void __launch_bounds__(512)
hidden_planes_kernel(const HiddenArgs a) {
  __shared__ float red[32];
  allow_dependents();
  dependency_wait();
  const long p = blockIdx.x;
  if (p >= a.counts[1]) return;
  const int e = a.ids[a.pair_of_pos[p]];
  const float* s1 = a.s1 + (size_t)e * 2 * a.I;
  const float as = a.ascale[p];
  const int splits = a.counts[2];
  float m = 0.f;
  for (int c = threadIdx.x * 4; c < a.I; c += blockDim.x * 4) {
    float h[4];
    hidden4(a, splits, p, s1, as, c, h);
    m = fmaxf(fmaxf(m, fmaxf(fabsf(h[0]), fabsf(h[1]))), fmaxf(fabsf(h[2]), fabsf(h[3])));
  }
  m = block_max(m, red);
  const float scale = __fdiv_rn(fmaxf(m, 1e-12f), 127.0f);
  const float inv = __fdiv_rn(1.0f, scale);
  if (threadIdx.x == 0) a.hscale[p] = scale;
  for (int c = threadIdx.x * 4; c < a.I; c += blockDim.x * 4) {
    float h[4];
    hidden4(a, splits, p, s1, as, c, h);
    *reinterpret_cast<uint32_t*>(a.hq + p * a.I + c) = quant4(h, scale, inv);
  }
}

// The hidden values and their rows' maxima are there: codes only.  A warp takes 32 * NV 16-byte vectors of a row, all of a
// lane's in flight together.
constexpr int kHiddenWarps = 8;
template <int NV>
__global__ void __launch_bounds__(32 * kHiddenWarps)
hidden_quant_kernel(const HiddenArgs a) {
  allow_dependents();
  dependency_wait();
  const int pieces = (a.I / 4 + 32 * NV - 1) / (32 * NV);
  const long task = (long)blockIdx.x * kHiddenWarps + (threadIdx.x >> 5);
  const long p = task / pieces;
  if (p >= a.rows) return;
  const int first = (int)(task - p * pieces) * 32 * NV + (threadIdx.x & 31);
  const float* src = a.h + p * a.I;
  uint4 raw[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i)
    raw[i] = first + 32 * i < a.I / 4 ? ld_stream_v4(src + 4 * (first + 32 * i)) : make_uint4(0u, 0u, 0u, 0u);
  const unsigned amax = a.amax[p];
  if (p >= a.counts[1]) return;   // (rows behind the last: requested like the others, so that no load waits for another)
  const float scale = __fdiv_rn(fmaxf(__uint_as_float(amax), 1e-12f), 127.0f);
  const float inv = __fdiv_rn(1.0f, scale);
  if (first == 0) a.hscale[p] = scale;
  uint32_t* dst = reinterpret_cast<uint32_t*>(a.hq + p * a.I);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    uint32_t out[1];
    quant_vec<float>(raw[i], scale, inv, out);
    if (first + 32 * i < a.I / 4) dst[first + 32 * i] = out[0];
  }
}

static int run_hidden(const HiddenArgs& a, cudaStream_t st) {
  // few rows are spread over many warps, many rows keep eight loads of a lane in flight (13332 rows of 1792: 42 -> 22 us against
  // CTAs of one row)
  const int nv = a.rows * (a.I / 4) > 4L * sm_count() * 2048 ? 8 : 1;
  const long tasks = a.rows * ((a.I / 4 + 32 * nv - 1) / (32 * nv));
  const dim3 grid((unsigned)((tasks + kHiddenWarps - 1) / kHiddenWarps)), block(32 * kHiddenWarps);
  const cudaError_t e = a.planes  ? launch_overlapped(hidden_planes_kernel, dim3((unsigned)a.rows), dim3(512), 0, st, a)
                        : nv == 8 ? launch_overlapped(hidden_quant_kernel<8>, grid, block, 0, st, a)
                                  : launch_overlapped(hidden_quant_kernel<1>, grid, block, 0, st, a);
  if (e != cudaSuccess) {
    record_cuda_error(e, "hidden rows launch");
    return LQ_ERR_CUDA;
  }
  return check_launch("hidden rows");
}

// ---------------------------------------------------------------------------------------------
// outputs from planes
// ---------------------------------------------------------------------------------------------
struct CombineArgs {
  const int32_t* planes;     // [splits][rows][N]
  const float* ascale;       // [rows]
  const float* s1;           // [E][N]
  const float* weights;      // [T][topk], or null: one output row per pair, unweighted
  const int* ids;            // [T][topk]
  const int* pos_of_pair;
  void* y;                   // [T][N] or [T * topk][N]
  long rows, outs;           // rows of a plane, rows of y
  const int* counts;         // of the plan: counts[2 + which] planes
  int N, topk, which, out_dtype;
};

// Four neighbouring outputs, at an offset that is a multiple of four.
__device__ __forceinline__ void store_out4(void* y, size_t at, const float (&v)[4], int out_dtype) {
  if (out_dtype == LQ_DT_F32) {
    *reinterpret_cast<float4*>(static_cast<float*>(y) + at) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    uint16_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) store_out(h, i, v[i], out_dtype);
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(y) + at) =
        make_uint2(h[0] | ((uint32_t)h[1] << 16), h[2] | ((uint32_t)h[3] << 16));
  }
}

// y = sum_j weight_j * (sums * row scale * channel scale), the experts of a token in the order of their slots, in float32,
// rounded once: products whose k was cut (few rows).  A thread makes VEC neighbouring channels; the rows' places, scales
// and weights are fetched by the lanes in parallel.  A chain of latencies (one token, 4096 channels: 4 us with its launch; the loads of two
// slots together were 0.2 us faster there and 1.2 us slower on 999 rows of 1024).
template <int VEC>
__global__ void __launch_bounds__(256)
combine_kernel(const CombineArgs a) {
  allow_dependents();
  dependency_wait();
  const int lane = threadIdx.x & 31;
  const int pieces = (a.N + 256 * VEC - 1) / (256 * VEC);
  const long m = blockIdx.x / pieces;
  const int c = ((int)(blockIdx.x - m * pieces) * 256 + threadIdx.x) * VEC;
  const int slots = a.weights ? a.topk : 1;
  const int splits = a.counts[2 + a.which];
  // lane j: slot j of the row
  int my_p = -1, my_e = 0;
  float my_scale = 0.f, my_w = 1.f;
  if (lane < slots) {
    my_p = a.pos_of_pair[m * slots + lane];
    my_e = a.ids[m * slots + lane];
    if (a.weights) my_w = a.weights[m * slots + lane];
    if (my_p >= 0) my_scale = a.ascale[my_p];
  }
  const bool in = c < a.N;   // the warp stays together for the shuffles
  float sum[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) sum[i] = 0.f;
  for (int j = 0; j < slots; ++j) {
    const int p = __shfl_sync(0xffffffffu, my_p, j), e = __shfl_sync(0xffffffffu, my_e, j);
    const float as = __shfl_sync(0xffffffffu, my_scale, j), w = __shfl_sync(0xffffffffu, my_w, j);
    if (p < 0 || !in) continue;
    const float* s1 = a.s1 + (size_t)e * a.N + c;
    float f[VEC];
    int v[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      f[i] = s1[i];
      v[i] = 0;
    }
#pragma unroll 4
    for (int s = 0; s < splits; ++s) {
      const int32_t* src = a.planes + ((size_t)s * a.rows + p) * a.N + c;
      if constexpr (VEC == 4) {
        const uint4 q = ld_stream_v4(src);
        v[0] += (int)q.x; v[1] += (int)q.y; v[2] += (int)q.z; v[3] += (int)q.w;
      } else {
        v[0] += src[0];
      }
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float o = lqq_scale(v[i], as, f[i]);
      sum[i] = a.weights ? __fmaf_rn(w, o, sum[i]) : o;
    }
  }
  if (!in) return;
  if constexpr (VEC == 4) store_out4(a.y, (size_t)m * a.N + c, sum, a.out_dtype);
  else store_out(a.y, (size_t)m * a.N + c, sum[0], a.out_dtype);
}

// The same weighted sum where the product wrote scaled rows in float32, one per pair in the tokens' order: the addresses
// are known at once, so all loads of a thread (four slots of IT * 4 channels) are in flight together; rows of pairs without an expert
// hold anything and are not used.  Bound by memory.  (From int32 sums in sorted order, each behind its pair's place, its row's scale
// and the channels' scales, which are as many bytes again out of L2: 8192 tokens x 2 x 4096 115 -> 60 us, 3333 x 4 x 4096
// 75 -> 43.)
template <int IT>
__global__ void __launch_bounds__(256)
weighted_sum_kernel(const float* rows, const float* weights, const int* ids, void* y, int E, int N, int topk, int out_dtype) {
  allow_dependents();
  dependency_wait();
  const int lane = threadIdx.x & 31;
  const int pieces = (N + 1024 * IT - 1) / (1024 * IT);
  const long m = blockIdx.x / pieces;
  const int c0 = ((int)(blockIdx.x - m * pieces) * 256 * IT + threadIdx.x) * 4;
  int my_e = -1;
  float my_w = 0.f;
  if (lane < topk) {
    my_e = ids[m * topk + lane];
    my_w = weights[m * topk + lane];
  }
  float sum[IT][4];
#pragma unroll
  for (int t = 0; t < IT; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[t][i] = 0.f;
  constexpr int kBatch = 4;
  for (int j0 = 0; j0 < topk; j0 += kBatch) {
    uint4 q[kBatch][IT];
#pragma unroll
    for (int b = 0; b < kBatch; ++b)
#pragma unroll
      for (int t = 0; t < IT; ++t)
        if (j0 + b < topk && c0 + 1024 * t < N) q[b][t] = ld_stream_v4(rows + (size_t)(m * topk + j0 + b) * N + c0 + 1024 * t);
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int e = __shfl_sync(0xffffffffu, my_e, (j0 + b) & 31);
      const float w = __shfl_sync(0xffffffffu, my_w, (j0 + b) & 31);
      if (j0 + b >= topk || e < 0 || e >= E) continue;   // (the whole warp)
#pragma unroll
      for (int t = 0; t < IT; ++t) {
        if (c0 + 1024 * t >= N) continue;
        sum[t][0] = __fmaf_rn(w, __uint_as_float(q[b][t].x), sum[t][0]);
        sum[t][1] = __fmaf_rn(w, __uint_as_float(q[b][t].y), sum[t][1]);
        sum[t][2] = __fmaf_rn(w, __uint_as_float(q[b][t].z), sum[t][2]);
        sum[t][3] = __fmaf_rn(w, __uint_as_float(q[b][t].w), sum[t][3]);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < IT; ++t)
    if (c0 + 1024 * t < N) store_out4(y, (size_t)m * N + c0 + 1024 * t, sum[t], out_dtype);
}

static int run_combine(const CombineArgs& a, cudaStream_t st) {
  const bool vec = a.N % 4 == 0 && (reinterpret_cast<uintptr_t>(a.y) & 15) == 0;
  const int piece = vec ? 1024 : 256;
  const dim3 grid((unsigned)(a.outs * ((a.N + piece - 1) / piece)));
  const cudaError_t e = vec ? launch_overlapped(combine_kernel<4>, grid, dim3(256), 0, st, a)
                            : launch_overlapped(combine_kernel<1>, grid, dim3(256), 0, st, a);
  if (e != cudaSuccess) {
    record_cuda_error(e, "combine_kernel launch");
    return LQ_ERR_CUDA;
  }
  return check_launch("combine_kernel");
}

// N a multiple of 4; rows and y 16-byte aligned.
static int run_weighted_sum(const float* rows, const float* weights, const int* ids, void* y, long T, int E, int N, int topk,
                            int out_dtype, cudaStream_t st) {
  const bool many = N > 1024 && T * (N / 1024) > 16L * sm_count();
  const int piece = many ? 2048 : 1024;
  const dim3 grid((unsigned)(T * ((N + piece - 1) / piece)));
  const cudaError_t e = many ? launch_overlapped(weighted_sum_kernel<2>, grid, dim3(256), 0, st, rows, weights, ids, y, E, N, topk, out_dtype)
                             : launch_overlapped(weighted_sum_kernel<1>, grid, dim3(256), 0, st, rows, weights, ids, y, E, N, topk, out_dtype);
  if (e != cudaSuccess) {
    record_cuda_error(e, "weighted_sum_kernel launch");
    return LQ_ERR_CUDA;
  }
  return check_launch("weighted_sum_kernel");
}

// ---------------------------------------------------------------------------------------------
// sizes
// ---------------------------------------------------------------------------------------------
// Rows of a tile, by what an expert gets on average (the router's choice is uneven: a tile holds twice that and more; ids that are no
// expert count too, since the host does not see them).  Measured with unevenly popular experts, tiles of 32 / 64 / 128 rows and the
// pair kernel, us; L: one product of 8 x 28672 x 4096, M, F: MLPs of 8 experts (4096, 14336) and of 16 (5120, 1536).
//   4-bit, rows:  8  L 89 / 88 / 100 / 122   M 129 / 131 / 148 / 183   F 54 / 56 / 62 / 67
//                12  L 84 / 81 / 92 / 108    M 142 / 137 / 159 / 191   F 57 / 61 / 67 / 67
//                32  L 129 / 111 / 114 / 148 M 214 / 188 / 187 / 220   F 70 / 65 / 69 / 70
//                48  L 176 / 124 / 118 / 137 M 274 / 194 / 195 / 229   F 86 / 69 / 79 / 76
//                64  L 216 / 146 / 137 / 154 M 337 / 256 / 215 / 233   F 103 / 74 / 83 / 80
//               128  L 363 / 211 / 180 / 192 M 584 / 385 / 341 / 292   F 163 / 126 / 122 / 112
//   INT8, whose operands need no unpacking:
//                 8  L 121 / 119 / 121 / 122 M 201 / 199 / 208 / 211   F 72 / 73 / 75 / 75
//                36  L 214 / 174 / 167 / 149 M 321 / 264 / 265 / 265   F 94 / 87 / 95 / 92
//                48  L 253 / 209 / 180 / 176 M 377 / 319 / 278 / 277   F 94 / 90 / 97 / 95
//                56  L 286 / 212 / 191 / 178 M 412 / 330 / 292 / 281   F 100 / 92 / 100 / 99
//               128  L 476 / 333 / 262 / 226 M 698 / 511 / 418 / 329   F 158 / 136 / 127 / 128
// The limits are where the forms cross on average over these, products of 64 x 2048 x 2048, 16 x 4096 x 4096, 32 x 4096 x 1792 and 64 x 1024 x
// 4096 and MLPs of 32 experts (4096, 1792), 64 (2048, 1024) and 128 (2048, 768); single layers are up to 10 % faster on the
// other side (4-bit from 96 to 127 rows the pair kernel is ahead on average, but up to 13 % behind where weights are small or experts few).
static int pick_bn(long pairs, int E, int w_kind) {
  const long mean = pairs / E;
  if (mean >= (w_kind == kBlob ? 128 : 45)) return w_kind == kBlob ? kPairRowsBlob : kPairRowsInt8;
  return mean <= 10 ? 32 : mean <= (w_kind == kBlob ? 48 : 40) ? 64 : 128;
}

// Whether a product's k may be cut, and into how many ranges at most, from the tiles that evenly chosen experts would make: where
// cutting shortens the time by a fifth (the planes are read again, by a pass behind the product), four k-steps a range at
// least, with room for twice the ranges in case the tokens choose fewer experts than that.  What may be cut has a few rounds of
// CTAs at most.
static SplitRule split_rule(long pairs, int E, int bn, int w_kind, int N, int K) {
  SplitRule r;
  r.n_tiles = (N + 127) / 128;
  r.kt = K / 128;
  r.most = 1;
  r.even = false;
  if (bn > 128) return r;   // the pair kernel takes whole tiles
  const long reached = pairs < E ? pairs : E;
  const long tiles = reached * ((pairs / reached + bn - 1) / bn);
  const int slots = 2 * sm_count(), room = K / 512 < 16 ? K / 512 : 16;
  int s = 1;
  if (tiles * r.n_tiles <= 8L * slots)
    for (int n = 2; n <= room; ++n)
      if (split_cost(tiles, r, n, slots) < split_cost(tiles, r, s, slots)) s = n;
  if (s > 1 && split_cost(tiles, r, s, slots) * 5 <= split_cost(tiles, r, 1, slots) * 4) r.most = 2 * s < room ? 2 * s : room;
  r.even = r.most == 1 && w_kind == kBlob && bn == kEvenRows && cut_evenly(tiles, r, slots);
  return r;
}

static size_t aligned(size_t bytes) { return (bytes + 255) & ~(size_t)255; }

// Takes pieces off a scratch buffer (or, with a null buffer, only counts them).
struct Carver {
  uint8_t* base;
  size_t used = 0;
  explicit Carver(void* p) : base(static_cast<uint8_t*>(p)) {}
  template <class T> T* take(size_t count) {
    T* p = base ? reinterpret_cast<T*>(base + used) : nullptr;
    used += aligned(count * sizeof(T));
    return p;
  }
};

// `N1`, `K1` and `N2`, `K2`: the products that use the plan (N2 = 0: one).
static Plan carve_plan(Carver& c, long pairs, int E, int w_kind, int N1, int K1, int N2, int K2) {
  Plan p;
  p.bn = pick_bn(pairs, E, w_kind);
  p.slots = 2 * sm_count();
  p.rule[0] = split_rule(pairs, E, p.bn, w_kind, N1, K1);
  p.rule[1] = N2 ? split_rule(pairs, E, p.bn, w_kind, N2, K2) : SplitRule{1, 1, 1, false};
  p.counts = c.take<int>(4);
  p.tiles = c.take<int4>((size_t)max_tiles(pairs, E, p.bn));
  p.pos_of_pair = c.take<int>((size_t)pairs);
  p.pair_of_pos = c.take<int>((size_t)pairs);
  for (int w = 0; w < 2; ++w) p.join[w] = p.rule[w].even ? c.take<int4>((size_t)p.slots) : nullptr;
  p.part = p.rule[0].even || p.rule[1].even ? c.take<int32_t>((size_t)p.slots * 2 * p.bn * 128) : nullptr;
  return p;
}

struct LinearBuffers {
  Plan plan;
  int8_t* xq;
  float* ascale;
  int32_t* planes;   // null: k stays whole
};
static LinearBuffers carve_linear(Carver& c, long pairs, int E, int N, int K, int w_kind) {
  LinearBuffers b;
  b.plan = carve_plan(c, pairs, E, w_kind, N, K, 0, 0);
  const int most = b.plan.rule[0].most;
  b.xq = c.take<int8_t>((size_t)pairs * K);
  b.ascale = c.take<float>((size_t)pairs);
  b.planes = most > 1 ? c.take<int32_t>((size_t)most * pairs * N) : nullptr;
  return b;
}

struct MlpBuffers {
  Plan plan;
  int8_t *xq, *hq;
  float *ascale, *hscale, *h;
  unsigned* amax;
  int32_t *planes1, *planes2;   // planes1 null: the product leaves h; planes2: the scaled rows where k stays whole
};
static MlpBuffers carve_mlp(Carver& c, long pairs, int E, int H, int I, int w_kind) {
  MlpBuffers b;
  b.plan = carve_plan(c, pairs, E, w_kind, 2 * I, H, H, I);
  const int most1 = b.plan.rule[0].most, most2 = b.plan.rule[1].most;
  b.xq = c.take<int8_t>((size_t)pairs * H);
  b.ascale = c.take<float>((size_t)pairs);
  b.hq = c.take<int8_t>((size_t)pairs * I);
  b.hscale = c.take<float>((size_t)pairs);
  b.planes1 = most1 > 1 ? c.take<int32_t>((size_t)most1 * pairs * 2 * I) : nullptr;
  b.h = most1 > 1 ? nullptr : c.take<float>((size_t)pairs * I);
  b.amax = most1 > 1 ? nullptr : c.take<unsigned>((size_t)pairs);
  b.planes2 = c.take<int32_t>((size_t)most2 * pairs * H);
  return b;
}

// Sizes that every call has to have; `N` rows and `K` columns of an expert's matrix.
static int check_sizes(long T, int topk, int E, int N, int K) {
  if (T < 1 || topk < 1 || E < 1 || N < 1 || K < 1) return LQ_ERR_BAD_ARG;
  if (topk > kMaxTopk || E > kMaxExperts || K % 128) return LQ_ERR_SHAPE;
  if (K >= 131072) return LQ_ERR_SHAPE;   // 2^17 products of -128 and -128 do not fit an int32 sum
  if (N >= 1 << 30) return LQ_ERR_SHAPE;  // the bytes of a row of 32-bit outputs are a 32-bit number
  if (T * topk > (1L << 24) || (long)E * ((N + 127) / 128 * 128) > 0x7fffffffL) return LQ_ERR_SHAPE;
  return LQ_OK;
}
static bool misaligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

}  // namespace experts
}  // namespace lq

using namespace lq;
using namespace lq::experts;

extern "C" {

int lq_moe_route(const void* logits, int logits_dtype, const float* bias, float* weights, int32_t* ids, int T, int E, int topk,
                 int scoring, int n_group, int topk_group, int group_score, int renormalize, float scale, void* stream) {
  if (!logits || !weights || !ids || T < 1 || E < 1 || topk < 1 || n_group < 1 || topk_group < 1) return LQ_ERR_BAD_ARG;
  if (logits_dtype < 0 || logits_dtype > LQ_DT_F32 || scoring < 0 || scoring > 1 || group_score < 0 || group_score > 1)
    return LQ_ERR_BAD_ARG;
  if (E > kMaxExperts || topk > kMaxTopk || E % n_group || topk_group > n_group || topk > topk_group * (E / n_group))
    return LQ_ERR_SHAPE;
  RouteArgs a;
  a.logits = logits;
  a.bias = bias;
  a.weights = weights;
  a.ids = ids;
  a.T = T;
  a.E = E;
  a.topk = topk;
  a.n_group = topk_group == n_group ? 1 : n_group;   // every group stays: nothing to rank
  a.topk_group = topk_group;
  a.group_size = (unsigned)(E / a.n_group);
  a.group_inv = ((1u << 20) + a.group_size - 1) / a.group_size;
  a.group_lanes = 1;
  while (2 * a.group_lanes * a.n_group <= 32) a.group_lanes *= 2;
  a.scale = scale;
  a.sigmoid = scoring == 1;
  a.top2 = group_score == 1;
  a.renormalize = renormalize != 0;
  cudaStream_t st = as_stream(stream);
  if (logits_dtype == LQ_DT_BF16) return launch_route<__nv_bfloat16>(a, st);
  if (logits_dtype == LQ_DT_F16) return launch_route<__half>(a, st);
  return launch_route<float>(a, st);
}

size_t lq_experts_linear_scratch_bytes(int T, int topk, int E, int N, int K, int w_kind) {
  if (w_kind < 0 || w_kind > 1) return 0;
  if (check_sizes(T, topk, E, N, K)) return 0;
  Carver c(nullptr);
  carve_linear(c, (long)T * topk, E, N, K, w_kind);
  return c.used;
}

int lq_experts_linear(const void* x, int x_dtype, const float* x_scale, int x_per_pair, const int32_t* ids, const void* w,
                      int w_kind, const float* s1, void* y, int out_dtype, int T, int topk, int E, int N, int K, void* scratch,
                      size_t scratch_bytes, void* stream) {
  if (!x || !ids || !w || !s1 || !y || x_dtype < 0 || x_dtype > 3 || (x_dtype == 3) != (x_scale != nullptr) || w_kind < 0 ||
      w_kind > 1 || out_dtype < 0 || out_dtype > LQ_DT_F32)
    return LQ_ERR_BAD_ARG;
  if (int rc = check_sizes(T, topk, E, N, K)) return rc;
  if (misaligned(x) || misaligned(w)) return LQ_ERR_SHAPE;
  Carver c(scratch);
  const long pairs = (long)T * topk;
  const LinearBuffers b = carve_linear(c, pairs, E, N, K, w_kind);
  if (!scratch || scratch_bytes < c.used || misaligned(scratch)) return LQ_ERR_WORKSPACE;
  cudaStream_t st = as_stream(stream);
  PlaceArgs pl = {};
  pl.x = x;
  pl.x_scale = x_scale;
  pl.xq = b.xq;
  pl.ascale = b.ascale;
  pl.y = b.planes ? nullptr : y;   // (from planes, the output pass writes every row)
  pl.y_size = out_dtype == LQ_DT_F32 ? 4 : 2;
  pl.per_row = x_per_pair ? 1 : topk;
  pl.K = K;
  pl.N = N;
  if (int rc = run_place(pl, ids, pairs, E, b.plan, x_dtype, x_per_pair ? pairs : T, st)) return rc;
  Product p = {};
  p.w = w;
  p.w_kind = w_kind;
  p.s1 = s1;
  p.x = b.xq;
  p.ascale = b.ascale;
  p.rows = pairs;
  p.E = E;
  p.N = N;
  p.K = K;
  p.which = 0;
  p.out_mode = b.planes ? kOutPlanes : kOutPairs;
  p.out_dtype = out_dtype;
  p.out = b.planes ? static_cast<void*>(b.planes) : y;
  if (int rc = run_product(p, b.plan, st)) return rc;
  if (!b.planes) return LQ_OK;
  CombineArgs k = {};
  k.planes = b.planes;
  k.ascale = b.ascale;
  k.s1 = s1;
  k.ids = ids;
  k.pos_of_pair = b.plan.pos_of_pair;
  k.y = y;
  k.rows = k.outs = pairs;
  k.N = N;
  k.topk = topk;
  k.counts = b.plan.counts;
  k.which = 0;
  k.out_dtype = out_dtype;
  return run_combine(k, st);
}

size_t lq_experts_mlp_scratch_bytes(int T, int topk, int E, int H, int I, int w_kind) {
  if (w_kind < 0 || w_kind > 1) return 0;
  if (check_sizes(T, topk, E, 2 * I, H) || check_sizes(T, topk, E, H, I)) return 0;
  Carver c(nullptr);
  carve_mlp(c, (long)T * topk, E, H, I, w_kind);
  return c.used;
}

int lq_experts_mlp(const void* x, int x_dtype, const float* weights, const int32_t* ids, const void* w13, const float* s13,
                   const void* w2, const float* s2, int w_kind, void* y, int out_dtype, int T, int topk, int E, int H, int I,
                   void* scratch, size_t scratch_bytes, void* stream) {
  if (!x || !weights || !ids || !w13 || !s13 || !w2 || !s2 || !y || x_dtype < 0 || x_dtype > LQ_DT_F32 || w_kind < 0 ||
      w_kind > 1 || out_dtype < 0 || out_dtype > LQ_DT_F32)
    return LQ_ERR_BAD_ARG;
  if (I > (1 << 29)) return LQ_ERR_SHAPE;
  if (int rc = check_sizes(T, topk, E, 2 * I, H)) return rc;
  if (int rc = check_sizes(T, topk, E, H, I)) return rc;
  if (misaligned(x) || misaligned(w13) || misaligned(w2) || misaligned(s13) || misaligned(s2) || misaligned(y)) return LQ_ERR_SHAPE;
  Carver c(scratch);
  const long pairs = (long)T * topk;
  const MlpBuffers b = carve_mlp(c, pairs, E, H, I, w_kind);
  if (!scratch || scratch_bytes < c.used || misaligned(scratch)) return LQ_ERR_WORKSPACE;
  cudaStream_t st = as_stream(stream);
  PlaceArgs pl = {};
  pl.x = x;
  pl.xq = b.xq;
  pl.ascale = b.ascale;
  pl.amax = b.amax;
  pl.per_row = topk;
  pl.K = H;
  if (int rc = run_place(pl, ids, pairs, E, b.plan, x_dtype, T, st)) return rc;
  Product p = {};
  p.w = w13;
  p.w_kind = w_kind;
  p.s1 = s13;
  p.x = b.xq;
  p.ascale = b.ascale;
  p.rows = pairs;
  p.E = E;
  p.N = 2 * I;
  p.K = H;
  p.which = 0;
  p.out_mode = b.planes1 ? kOutPlanes : kOutGated;
  p.out = b.planes1 ? static_cast<void*>(b.planes1) : b.h;
  p.amax = b.amax;
  if (int rc = run_product(p, b.plan, st)) return rc;
  HiddenArgs h = {};
  h.planes = b.planes1;
  h.h = b.h;
  h.amax = b.amax;
  h.ascale = b.ascale;
  h.s1 = s13;
  h.ids = ids;
  h.counts = b.plan.counts;
  h.pair_of_pos = b.plan.pair_of_pos;
  h.hq = b.hq;
  h.hscale = b.hscale;
  h.rows = pairs;
  h.I = I;
  if (int rc = run_hidden(h, st)) return rc;
  p.w = w2;
  p.s1 = s2;
  p.x = b.hq;
  p.ascale = b.hscale;
  p.N = H;
  p.K = I;
  p.which = 1;
  if (b.plan.rule[1].most == 1) {
    // whole k-ranges: scaled rows in the tokens' order, in the bytes of one plane
    p.out_mode = kOutPairs;
    p.out_dtype = LQ_DT_F32;
    p.out = b.planes2;
    if (int rc = run_product(p, b.plan, st)) return rc;
    return run_weighted_sum(reinterpret_cast<const float*>(b.planes2), weights, ids, y, T, E, H, topk, out_dtype, st);
  }
  p.out_mode = kOutPlanes;
  p.out = b.planes2;
  if (int rc = run_product(p, b.plan, st)) return rc;
  CombineArgs k = {};
  k.planes = b.planes2;
  k.ascale = b.hscale;
  k.s1 = s2;
  k.weights = weights;
  k.ids = ids;
  k.pos_of_pair = b.plan.pos_of_pair;
  k.y = y;
  k.rows = pairs;
  k.outs = T;
  k.N = H;
  k.topk = topk;
  k.counts = b.plan.counts;
  k.which = 1;
  k.out_dtype = out_dtype;
  return run_combine(k, st);
}

}  // extern "C"
