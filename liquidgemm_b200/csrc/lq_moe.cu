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
// Where scores decide what is chosen (keys with a bias, sums of two) they are worked out in float64: neighbouring keys may
// lie closer than a float32 exponential's error, and a choice is a whole number.
// A logit of -inf or NaN, or a bias that makes a key so, takes its expert out.
//
// Bound by instruction issue (a token's row is a few hundred bytes).  A choice is one 32-bit warp reduction over the keys'
// upper halves and a ballot; the lower halves and the indices are compared only where several lanes hold the same upper half.
// Groups are ranked from shared memory, 32 / G lanes to a group.  (A warp reduction of the 64-bit key for every group and
// choice, as in the first form: 8192 tokens, 192 experts in 8 groups, 64 us.)

// Orders numbers like unsigned integers; every number's image is above 0, which stands for "not to be chosen".
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t u = __float_as_uint(v + 0.0f);   // -0 becomes 0: equal keys are equal bits
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ unsigned long long ordered(double v) {
  const unsigned long long u = (unsigned long long)__double_as_longlong(v + 0.0);
  return u ^ ((u >> 63) ? 0xffffffffffffffffull : 0x8000000000000000ull);
}
__device__ __forceinline__ uint32_t upper(uint32_t k) { return k; }
__device__ __forceinline__ uint32_t upper(unsigned long long k) { return (uint32_t)(k >> 32); }
__device__ __forceinline__ uint32_t lower(uint32_t) { return 0u; }
__device__ __forceinline__ uint32_t lower(unsigned long long k) { return (uint32_t)k; }

struct RouteArgs {
  const void* logits;
  const float* bias;
  float* weights;
  int* ids;
  int T, E, topk, n_group, topk_group;
  float scale;
  bool sigmoid, top2, renormalize;
};

template <typename S> struct KeyOf;
template <> struct KeyOf<float> { using type = uint32_t; };
template <> struct KeyOf<double> { using type = unsigned long long; };

constexpr int kRouteWarps = 4;

// Which groups stay: true for the groups of the topk_group highest ranks, the lowest index among equals.  `v` [E]: what the
// groups are ranked by, -inf where an expert cannot be chosen; `rank` [n_group] and `kept` [n_group] are this warp's.
template <typename S>
__device__ __forceinline__ void rank_groups(const RouteArgs& a, const S* v, S* rank, uint8_t* kept) {
  const int lane = threadIdx.x & 31;
  const int G = a.n_group, size = a.E / G;
  int L = 1;   // lanes of a group
  while (2 * L * G <= 32) L *= 2;
  for (int base = 0; base < G; base += 32 / L) {
    const int g = base + lane / L;
    S m1 = -INFINITY, m2 = -INFINITY;
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
    if (g < G && (lane & (L - 1)) == 0) rank[g] = a.top2 && m2 > (S)-INFINITY ? m1 + m2 : m1;
  }
  __syncwarp();
  for (int g = lane; g < G; g += 32) {
    const S mine = rank[g];
    int before = 0;
    for (int o = 0; o < G; ++o) before += (rank[o] > mine || (rank[o] == mine && o < g)) ? 1 : 0;
    kept[g] = before < a.topk_group;
  }
  __syncwarp();
}

// S: the type of the scores (and with a bias of the keys).
template <typename T, int PER, typename S>
__global__ void __launch_bounds__(32 * kRouteWarps)
route_kernel(const RouteArgs a) {
  using Key = typename KeyOf<S>::type;
  __shared__ S values[kRouteWarps][PER * 32];
  __shared__ S ranks[kRouteWarps][PER * 32];
  __shared__ uint8_t kept[kRouteWarps][PER * 32];
  allow_dependents();
  dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long t = (long)blockIdx.x * kRouteWarps + warp;
  if (t >= a.T) return;
  const T* row = static_cast<const T*>(a.logits) + t * a.E;
  const float none = -INFINITY;
  float l[PER];
  float top = none;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = lane + 32 * i;
    l[i] = e < a.E ? to_f32<T>(row[e]) : none;
    if (!(l[i] > none)) l[i] = none;   // NaN too
    top = fmaxf(top, l[i]);
  }

  S s[PER];
  if (a.sigmoid) {
#pragma unroll
    for (int i = 0; i < PER; ++i) s[i] = l[i] > none ? (S)1 / ((S)1 + exp(-(S)l[i])) : (S)0;
  } else {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    S sum = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      s[i] = !(l[i] > none) ? (S)0 : l[i] == top ? (S)1 : exp((S)l[i] - (S)top);   // (equal to the largest: also where that is infinite)
      sum += s[i];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const S d = sum > 0 ? sum : (S)1;
#pragma unroll
    for (int i = 0; i < PER; ++i) s[i] = s[i] / d;
  }

  const bool by_score = a.bias != nullptr;
  Key key[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = lane + 32 * i;
    S v = (S)none;
    if (l[i] > none) v = by_score ? s[i] + (S)a.bias[e] : (S)l[i];
    const bool can = v > (S)none;   // (false for NaN)
    key[i] = can ? ordered(v) : 0;
    if (a.n_group > 1) values[warp][e] = !can ? (S)none : a.top2 && !by_score ? s[i] : v;
  }
  if (a.n_group > 1) {
    __syncwarp();
    rank_groups<S>(a, values[warp], ranks[warp], kept[warp]);
    const unsigned size = a.E / a.n_group, inv = ((1u << 20) + size - 1) / size;   // e / size for e < 512
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const unsigned e = lane + 32 * i;
      if (e < a.E && !kept[warp][e * inv >> 20]) key[i] = 0;
    }
  }

  // lane j ends up with choice j
  int my_id = -1;
  S my_w = 0;
  Key mine = 0;
  int at = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (key[i] > mine) mine = key[i], at = i;
  for (int j = 0; j < a.topk; ++j) {
    const uint32_t best = __reduce_max_sync(0xffffffffu, upper(mine));
    if (best == 0) break;   // (no key's upper half is 0)
    unsigned who = __ballot_sync(0xffffffffu, upper(mine) == best);
    if (who & (who - 1)) {   // several lanes: the lower halves, then the index
      const bool in = upper(mine) == best;
      const uint32_t low = __reduce_max_sync(0xffffffffu, in ? lower(mine) : 0u);
      const unsigned first = __reduce_min_sync(0xffffffffu, in && lower(mine) == low ? (unsigned)(lane + 32 * at) : 1u << 20);
      who = 1u << (first & 31);
    }
    const int owner = __ffs(who) - 1;
    const int id = __shfl_sync(0xffffffffu, lane + 32 * at, owner);
    S w = 0;
    if (lane == owner) {
      mine = 0;
      const int gone = at;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        if (i == gone) key[i] = 0, w = s[i];
        if (key[i] > mine) mine = key[i], at = i;
      }
    }
    w = __shfl_sync(0xffffffffu, w, owner);
    if (lane == j) my_id = id, my_w = w;
  }
  if (a.renormalize) {
    S total = my_w;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    if (total > 0) my_w = my_w / total;
  }
  if (lane < a.topk) {
    a.weights[t * a.topk + lane] = (float)(my_w * (S)a.scale);
    a.ids[t * a.topk + lane] = my_id;
  }
}

template <typename T, typename S>
static int launch_route(const RouteArgs& a, cudaStream_t st) {
  const int per = (a.E + 31) / 32;
  void (*kern)(RouteArgs) = per <= 1    ? route_kernel<T, 1, S>
                            : per <= 2  ? route_kernel<T, 2, S>
                            : per <= 4  ? route_kernel<T, 4, S>
                            : per <= 6  ? route_kernel<T, 6, S>
                            : per <= 8  ? route_kernel<T, 8, S>
                            : per <= 12 ? route_kernel<T, 12, S>
                                        : route_kernel<T, 16, S>;
  const cudaError_t e = launch_overlapped(kern, dim3((a.T + kRouteWarps - 1) / kRouteWarps), dim3(32 * kRouteWarps), 0, st, a);
  if (e != cudaSuccess) {
    record_cuda_error(e, "route_kernel launch");
    return LQ_ERR_CUDA;
  }
  return check_launch("route_kernel");
}

// ---------------------------------------------------------------------------------------------
// plan
// ---------------------------------------------------------------------------------------------
// The tiles of expert e: as few as cover its n rows, and of equal widths in steps of 32 (a full tile and a narrow rest would
// take as long as two full ones wherever the two run side by side).  Every one has a row: bn is a multiple of 32.
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
// on every run.
constexpr int kPlanWarps = 32;
__global__ void __launch_bounds__(32 * kPlanWarps)
plan_kernel(const int* ids, long pairs, int E, const Plan plan) {
  extern __shared__ int hist[];   // [kPlanWarps][E]
  __shared__ int sums[2][kPlanWarps];
  allow_dependents();
  dependency_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < kPlanWarps * E; i += blockDim.x) hist[i] = 0;
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
  if (e < E) {
    for (int w = 0; w < kPlanWarps; ++w) {
      const int c = hist[w * E + e];
      hist[w * E + e] = n;
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
    for (int w = 0; w < kPlanWarps; ++w) hist[w * E + e] += row0;
    write_tiles(plan, tile0, e, row0, n, tiles);
  }
  if (threadIdx.x == blockDim.x - 1) {
    plan.counts[0] = rb + b;
    plan.counts[1] = ra + a;
  }
  __syncthreads();
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
      const unsigned same = __match_any_sync(0xffffffffu, id[q]);
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
// Up to kSortedHere pairs (`plan.tiles` set) there is no plan kernel before this one: a CTA finds the places of its own pairs
// by counting the pairs that come before them, and one more CTA (the first) cuts the experts' rows into tiles.  That
// saves a launch and its hand-over, 4 of the 9 us before the first product of a decode step; the counting grows with
// the square of the pairs (at 2048 it takes the time of the plan kernel).
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
  const int* ids;          // with plan.tiles: the sort is done here
  int pairs, E;
  Plan plan;
};

// Tiles and counts of the plan (one CTA of any size).
__device__ __forceinline__ void make_tiles(const PlaceArgs& a) {
  __shared__ int hist[kMaxExperts];
  for (int e = threadIdx.x; e < kMaxExperts; e += blockDim.x) hist[e] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < a.pairs; i += blockDim.x) {
    const int e = a.ids[i];
    if (e >= 0 && e < a.E) atomicAdd(&hist[e], 1);
  }
  __syncthreads();
  if (threadIdx.x >= 32) return;
  constexpr int kPer = kMaxExperts / 32;   // neighbouring experts of a lane
  const int lane = threadIdx.x;
  int rows = 0, tiles = 0;
#pragma unroll
  for (int q = 0; q < kPer; ++q) {
    const int n = hist[lane * kPer + q];
    rows += n;
    tiles += (n + a.plan.bn - 1) / a.plan.bn;
  }
  int r = rows, t = tiles;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int pr = __shfl_up_sync(0xffffffffu, r, o), pt = __shfl_up_sync(0xffffffffu, t, o);
    if (lane >= o) r += pr, t += pt;
  }
  if (lane == 31) {
    a.plan.counts[0] = t;
    a.plan.counts[1] = r;
  }
  r -= rows;
  t -= tiles;
  for (int q = 0; q < kPer; ++q) {
    const int e = lane * kPer + q, n = hist[e];
    const int mine = (n + a.plan.bn - 1) / a.plan.bn;
    write_tiles(a.plan, t, e, r, n, mine);
    t += mine;
    r += n;
  }
}

// The places of the pairs of row m, in `place` [per_row] (shared memory): read from the plan, or counted and entered there.
__device__ __forceinline__ void find_places(const PlaceArgs& a, long m, int* place) {
  if (!a.plan.tiles) {
    for (int j = threadIdx.x; j < a.per_row; j += blockDim.x) place[j] = a.pos_of_pair[m * a.per_row + j];
  } else {
    const int lane = threadIdx.x & 31;
    for (int j = threadIdx.x >> 5; j < a.per_row; j += blockDim.x >> 5) {
      const int pair = (int)m * a.per_row + j;
      const int e = a.ids[pair];
      int before = 0;
#pragma unroll 4
      for (int i = lane; i < a.pairs; i += 32) {
        const int o = a.ids[i];
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

template <typename T, int NV>
__global__ void __launch_bounds__(1024)
place_rows_kernel(const PlaceArgs a) {
  __shared__ float red[32];
  __shared__ int place[kMaxTopk];
  constexpr int VEC = 16 / sizeof(T);
  allow_dependents();
  dependency_wait();
  if (a.plan.tiles && blockIdx.x == 0) {
    make_tiles(a);
    return;
  }
  const long m = a.plan.tiles ? blockIdx.x - 1 : blockIdx.x;
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
  find_places(a, m, place);
  const float amax = block_max(rm.value(), red);   // (its barrier orders the places too)
  const float scale = __fdiv_rn(fmaxf(amax, 1e-12f), 127.0f);
  const float inv = __fdiv_rn(1.0f, scale);
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
    int8_t* qr = a.xq + (long)p * a.K;
    if constexpr (NV > 0) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = threadIdx.x + i * blockDim.x;
        if (v >= nvec) break;
        uint32_t out[4 / sizeof(T)];
        quant_vec<T>(raw[i], scale, inv, out);
        if constexpr (sizeof(T) == 4) reinterpret_cast<uint32_t*>(qr)[v] = out[0];
        else reinterpret_cast<uint2*>(qr)[v] = make_uint2(out[0], out[1]);
      }
    } else {
      for (int v = threadIdx.x; v < nvec; v += blockDim.x) {
        uint32_t out[4 / sizeof(T)];
        quant_vec<T>(xr[v], scale, inv, out);
        if constexpr (sizeof(T) == 4) reinterpret_cast<uint32_t*>(qr)[v] = out[0];
        else reinterpret_cast<uint2*>(qr)[v] = make_uint2(out[0], out[1]);
      }
    }
  }
}

// Rows that come in INT8 with their scales.
__global__ void __launch_bounds__(256)
place_i8_kernel(const PlaceArgs a) {
  __shared__ int place[kMaxTopk];
  allow_dependents();
  dependency_wait();
  if (a.plan.tiles && blockIdx.x == 0) {
    make_tiles(a);
    return;
  }
  const long m = a.plan.tiles ? blockIdx.x - 1 : blockIdx.x;
  find_places(a, m, place);
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

template <typename T>
static int launch_place(const PlaceArgs& a, long rows, cudaStream_t st) {
  int threads = 0;
  const int nv = row_units_per_thread(rows, a.K / (16 / (int)sizeof(T)), 8, 128, 1024, &threads);
  void (*kern)(PlaceArgs) = nv == 1   ? place_rows_kernel<T, 1>
                            : nv == 2 ? place_rows_kernel<T, 2>
                            : nv == 4 ? place_rows_kernel<T, 4>
                            : nv == 8 ? place_rows_kernel<T, 8>
                                      : place_rows_kernel<T, 0>;
  if (nv == 0) threads = 1024;
  const cudaError_t e = launch_overlapped(kern, dim3((unsigned)rows + (a.plan.tiles ? 1u : 0u)), dim3(threads), 0, st, a);
  if (e != cudaSuccess) {
    record_cuda_error(e, "place_rows_kernel launch");
    return LQ_ERR_CUDA;
  }
  return check_launch("place_rows_kernel");
}

// Plan and rows.
static int run_place(PlaceArgs& a, const int* ids, long pairs, int E, const Plan& plan, int x_dtype, long rows, cudaStream_t st) {
  a.pos_of_pair = plan.pos_of_pair;
  if (pairs <= kSortedHere) {
    a.ids = ids;
    a.pairs = (int)pairs;
    a.E = E;
    a.plan = plan;
  } else if (int rc = run_plan(ids, pairs, E, plan, st)) {
    return rc;
  }
  if (x_dtype == LQ_DT_BF16) return launch_place<__nv_bfloat16>(a, rows, st);
  if (x_dtype == LQ_DT_F16) return launch_place<__half>(a, rows, st);
  if (x_dtype == LQ_DT_F32) return launch_place<float>(a, rows, st);
  const cudaError_t e = launch_overlapped(place_i8_kernel, dim3((unsigned)rows + (a.plan.tiles ? 1u : 0u)), dim3(256), 0, st, a);
  if (e != cudaSuccess) {
    record_cuda_error(e, "place_i8_kernel launch");
    return LQ_ERR_CUDA;
  }
  return check_launch("place_i8_kernel");
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
  int I, splits;
};

// Four hidden values of row p from the planes.
__device__ __forceinline__ void hidden4(const HiddenArgs& a, long p, const float* s1, float as, int c, float (&h)[4]) {
  int4 g0 = make_int4(0, 0, 0, 0), g1 = g0;
  for (int s = 0; s < a.splits; ++s) {
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
// second pass finds in L2.
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
  float m = 0.f;
  for (int c = threadIdx.x * 4; c < a.I; c += blockDim.x * 4) {
    float h[4];
    hidden4(a, p, s1, as, c, h);
    m = fmaxf(fmaxf(m, fmaxf(fabsf(h[0]), fabsf(h[1]))), fmaxf(fabsf(h[2]), fabsf(h[3])));
  }
  m = block_max(m, red);
  const float scale = __fdiv_rn(fmaxf(m, 1e-12f), 127.0f);
  const float inv = __fdiv_rn(1.0f, scale);
  if (threadIdx.x == 0) a.hscale[p] = scale;
  for (int c = threadIdx.x * 4; c < a.I; c += blockDim.x * 4) {
    float h[4];
    hidden4(a, p, s1, as, c, h);
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
  int N, topk, splits, out_dtype;
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
// and weights are fetched by the lanes in parallel.
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
    for (int s = 0; s < a.splits; ++s) {
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
// Rows of a tile: what an expert gets on average, with room for the uneven choice of a router.
static int pick_bn(long pairs, int E, int w_kind) {
  const long mean = pairs / E;
  if (mean >= 96) return w_kind == kBlob ? kPairRowsBlob : kPairRowsInt8;
  return mean <= 12 ? 32 : mean <= 40 ? 64 : 128;
}

// K-ranges of a product: only where the tiles of the experts that can be reached leave half of the CTA slots free, and with four
// k-steps a range at least.
static int pick_splits(long pairs, int E, int bn, int N, int K) {
  if (bn > 128) return 1;   // the pair kernel takes whole tiles
  const long reached = pairs < E ? pairs : E;
  const long tiles = reached * ((pairs / reached + bn - 1) / bn) * ((N + 127) / 128);
  const long slots = 2L * sm_count();
  int S = (int)(slots / tiles);
  if (S > K / 512) S = K / 512;
  if (S > 16) S = 16;
  return S < 1 ? 1 : S;
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

static Plan carve_plan(Carver& c, long pairs, int E, int w_kind) {
  Plan p;
  p.bn = pick_bn(pairs, E, w_kind);
  p.counts = c.take<int>(4);
  p.tiles = c.take<int4>((size_t)max_tiles(pairs, E, p.bn));
  p.pos_of_pair = c.take<int>((size_t)pairs);
  p.pair_of_pos = c.take<int>((size_t)pairs);
  return p;
}

struct LinearBuffers {
  Plan plan;
  int8_t* xq;
  float* ascale;
  int32_t* planes;
  int splits;
};
static LinearBuffers carve_linear(Carver& c, long pairs, int E, int N, int K, int w_kind) {
  LinearBuffers b;
  b.plan = carve_plan(c, pairs, E, w_kind);
  b.splits = pick_splits(pairs, E, b.plan.bn, N, K);
  b.xq = c.take<int8_t>((size_t)pairs * K);
  b.ascale = c.take<float>((size_t)pairs);
  b.planes = b.splits > 1 ? c.take<int32_t>((size_t)b.splits * pairs * N) : nullptr;
  return b;
}

struct MlpBuffers {
  Plan plan;
  int8_t *xq, *hq;
  float *ascale, *hscale, *h;
  unsigned* amax;
  int32_t *planes1, *planes2;
  int splits1, splits2;
};
static MlpBuffers carve_mlp(Carver& c, long pairs, int E, int H, int I, int w_kind) {
  MlpBuffers b;
  b.plan = carve_plan(c, pairs, E, w_kind);
  b.splits1 = pick_splits(pairs, E, b.plan.bn, 2 * I, H);
  b.splits2 = pick_splits(pairs, E, b.plan.bn, H, I);
  b.xq = c.take<int8_t>((size_t)pairs * H);
  b.ascale = c.take<float>((size_t)pairs);
  b.hq = c.take<int8_t>((size_t)pairs * I);
  b.hscale = c.take<float>((size_t)pairs);
  b.planes1 = b.splits1 > 1 ? c.take<int32_t>((size_t)b.splits1 * pairs * 2 * I) : nullptr;
  b.h = b.splits1 > 1 ? nullptr : c.take<float>((size_t)pairs * I);
  b.amax = b.splits1 > 1 ? nullptr : c.take<unsigned>((size_t)pairs);
  b.planes2 = c.take<int32_t>((size_t)b.splits2 * pairs * H);
  return b;
}

// Sizes that every call has to have; `N` rows and `K` columns of an expert's matrix.
static int check_sizes(long T, int topk, int E, int N, int K) {
  if (T < 1 || topk < 1 || E < 1 || N < 1 || K < 1) return LQ_ERR_BAD_ARG;
  if (topk > kMaxTopk || E > kMaxExperts || K % 128) return LQ_ERR_SHAPE;
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
  a.scale = scale;
  a.sigmoid = scoring == 1;
  a.top2 = group_score == 1;
  a.renormalize = renormalize != 0;
  // (sigmoid scores far below 1 would lose their ratio in float32's denormal range)
  const bool wide = a.sigmoid || bias != nullptr || (a.n_group > 1 && a.top2);
  cudaStream_t st = as_stream(stream);
  if (logits_dtype == LQ_DT_BF16) return wide ? launch_route<__nv_bfloat16, double>(a, st) : launch_route<__nv_bfloat16, float>(a, st);
  if (logits_dtype == LQ_DT_F16) return wide ? launch_route<__half, double>(a, st) : launch_route<__half, float>(a, st);
  return wide ? launch_route<float, double>(a, st) : launch_route<float, float>(a, st);
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
  p.splits = b.splits;
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
  k.splits = b.splits;
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
  p.splits = b.splits1;
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
  h.splits = b.splits1;
  if (int rc = run_hidden(h, st)) return rc;
  p.w = w2;
  p.s1 = s2;
  p.x = b.hq;
  p.ascale = b.hscale;
  p.N = H;
  p.K = I;
  p.splits = b.splits2;
  if (b.splits2 == 1) {
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
  k.splits = b.splits2;
  k.out_dtype = out_dtype;
  return run_combine(k, st);
}

}  // extern "C"
