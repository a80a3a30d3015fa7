// Low-rank adapters of many requests at once, added to a projection's output:
//   v[t, s, j] = sum_k A[l, s, j, k] x[t, k]                                 l = ids[t], float32
//   out[t, n]  = (type of y)(y[t, n] + scale[l] * sum_j B[l, n, j] v[t, slice of n, j])
// Three kernels: rows are put in the order of their adapters and cut into tiles of up to 64 rows of one adapter; a tile's rows
// times A (K cut over warps and CTAs); the result times B, added to y.  The rows that a slot gets are known on the device only.
#include "lq_common.cuh"

namespace lq {
namespace {

constexpr int kTile = 64;            // rows of a tile, at most
constexpr int kMaxSlices = 8;
constexpr int kMaxSlots = 4096;
constexpr int kMaxRank = 256;
constexpr int kMaxSplits = 16;

// A tile: `count` rows order[start ...] of slot `slot`; slot -1: rows to copy.  count 0: no tile.
struct Tile {
  int slot, start, count, pad;
};

struct Slices {
  int n;
  int start[kMaxSlices + 1];   // first column of a slice
  int block[kMaxSlices + 1];   // first column block of a slice (blocks end with their slice)
};

template <typename T> struct Mma;
template <> struct Mma<__nv_bfloat16> {
  static __device__ __forceinline__ void run(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <> struct Mma<__half> {
  static __device__ __forceinline__ void run(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

template <typename T> __device__ __forceinline__ T narrow(float v);
template <> __device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ float narrow<float>(float v) { return v; }

// Coherent loads that may stay in L1 (other warps or tiles read the same weights).
__device__ __forceinline__ uint4 ld_v4(const void* p) {
  uint4 r;
  asm volatile("ld.global.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p) : "memory");
  return r;
}
__device__ __forceinline__ uint2 ld_v2(const void* p) {
  uint2 r;
  asm volatile("ld.global.v2.u32 {%0,%1}, [%2];" : "=r"(r.x), "=r"(r.y) : "l"(p) : "memory");
  return r;
}

// The slot of a row, L where it has none (an id outside the slots, a slot without any slice's matrices).
__device__ __forceinline__ int slot_of(const void* ids, bool wide, long t, int L, int S, const int* rank) {
  const long id = wide ? static_cast<const long long*>(ids)[t] : static_cast<const int*>(ids)[t];
  bool any = false;
  if (id >= 0 && id < L)
    for (int s = 0; s < S; ++s) any |= rank[id * S + s] > 0;
  return any ? (int)id : L;
}

// ---------------------------------------------------------------------------------------------
// Rows in the order of their slots, tiles.  One CTA.  The order within a slot hangs on atomics; no result does, since a row's sums
// are its own wherever it lies in a tile.
__global__ void __launch_bounds__(1024)
adapter_plan_kernel(const void* ids, bool wide, const int* rank, int T, int L, int S, bool copy_rest, int* order, Tile* tiles,
                    int max_tiles) {
  extern __shared__ int smem[];
  int* first = smem;                  // [L + 2] rows before a slot's
  int* tile0 = smem + L + 2;          // [L + 2] tiles before a slot's
  int* next = tile0 + L + 2;          // [L + 1] counts, then the next free place
  __shared__ int warp_sum[2][32];
  allow_dependents();
  dependency_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int i = tid; i <= L; i += blockDim.x) next[i] = 0;
  __syncthreads();
  for (int t0 = warp * 32; t0 < T; t0 += blockDim.x) {
    const int t = t0 + lane;
    const int b = t < T ? slot_of(ids, wide, t, L, S, rank) : -1;
    const unsigned same = __match_any_sync(0xffffffffu, b);
    if (b >= 0 && lane == __ffs(same) - 1) atomicAdd(&next[b], __popc(same));
  }
  __syncthreads();
  // exclusive sums over the slots, a run of neighbours per thread
  const int per = (L + 1 + blockDim.x - 1) / blockDim.x, lo = min(L + 1, tid * per), hi = min(L + 1, lo + per);
  int rows = 0, cut = 0;
  for (int i = lo; i < hi; ++i) {
    rows += next[i];
    if (i < L || copy_rest) cut += (next[i] + kTile - 1) / kTile;
  }
  int r = rows, c = cut;
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, r, o), b = __shfl_up_sync(0xffffffffu, c, o);
    if (lane >= o) r += a, c += b;
  }
  if (lane == 31) warp_sum[0][warp] = r, warp_sum[1][warp] = c;
  __syncthreads();
  for (int w = 0; w < warp; ++w) r += warp_sum[0][w], c += warp_sum[1][w];
  r -= rows, c -= cut;
  for (int i = lo; i < hi; ++i) {
    const int n = next[i];
    first[i] = r, tile0[i] = c, next[i] = r;
    r += n;
    if (i < L || copy_rest) c += (n + kTile - 1) / kTile;
    if (i == L) first[L + 1] = r, tile0[L + 1] = c;
  }
  __syncthreads();
  for (int i = tid; i < max_tiles; i += blockDim.x) {
    Tile tile = {-1, 0, 0, 0};
    if (i < tile0[L + 1]) {
      int a = 0, b = L + 1;   // the last slot whose tiles begin at or before i (those without tiles begin where the next does)
      while (b - a > 1) {
        const int mid = (a + b) / 2;
        if (tile0[mid] <= i) a = mid;
        else b = mid;
      }
      const int at = first[a] + (i - tile0[a]) * kTile;
      tile = {a == L ? -1 : a, at, min(kTile, first[a + 1] - at), 0};
    }
    tiles[i] = tile;
  }
  for (int t0 = warp * 32; t0 < T; t0 += blockDim.x) {
    const int t = t0 + lane;
    const int b = t < T ? slot_of(ids, wide, t, L, S, rank) : -1;
    const unsigned same = __match_any_sync(0xffffffffu, b);
    const int leader = __ffs(same) - 1;
    int at = 0;
    if (b >= 0 && lane == leader) at = atomicAdd(&next[b], __popc(same));
    at = __shfl_sync(0xffffffffu, at, leader) + __popc(same & ((1u << lane) - 1));
    if (b >= 0) order[at] = t;
  }
}

// ---------------------------------------------------------------------------------------------
// v = A x for a tile's rows: ranks are the 16 rows of an MMA, eight tokens its columns, so that both operands come straight
// from their row-major matrices into registers.  The order of k within a product is free: thread t of a quad takes the
// eight neighbours 8 t .. 8 t + 7 of 32 k for both operands, one 16-byte load each.  A CTA's warps take turns at the 32-k
// chunks of its range of K; their sums meet in shared memory and go to plane blockIdx.z of v [planes][T][R] (R = slices x stack
// rank), in the order of the plan.
template <typename T, int RT>
__global__ void __launch_bounds__(256, 1)
adapter_shrink_kernel(const T* x, long ldx, const T* a, const int* rank, const int* order, const Tile* tiles, float* v, int rows,
                      int K, int R, int rp, int k_range) {
  extern __shared__ float part[];   // [8 warps][RT * 16][66]
  __shared__ int row_of[kTile];
  constexpr int kPitch = 66;
  allow_dependents();
  dependency_wait();
  const Tile tile = tiles[blockIdx.x];
  if (tile.count == 0 || tile.slot < 0) return;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  if (tid < kTile) row_of[tid] = order[tile.start + min(tid, tile.count - 1)];
  const int r0 = blockIdx.y * (RT * 16), S = R / rp;
  const int k0 = blockIdx.z * k_range, k1 = min(K, k0 + k_range);
  const T* al = a + (long)tile.slot * R * K;
  bool live[RT][2];   // the eight-row halves of the rank tiles that the slices' ranks reach (rp % 8 == 0)
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = r0 + i * 16 + h * 8;
      live[i][h] = r < R && r % rp < rank[tile.slot * S + r / rp];
    }
  const int tokens8 = (tile.count + 7) / 8;
  float acc[RT][8][4];
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[i][j][0] = acc[i][j][1] = acc[i][j][2] = acc[i][j][3] = 0.f;
  __syncthreads();
  for (int k = k0 + warp * 32; k < k1; k += 256) {
    const int kk = k + 8 * t;
    const bool in = kk < k1;
    uint4 xa[8], aa[RT][2];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      xa[j] = in && j < tokens8 ? ld_stream_v4(x + (long)row_of[j * 8 + g] * ldx + kk) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        aa[i][h] = in && live[i][h] ? ld_v4(al + (long)(r0 + i * 16 + h * 8 + g) * K + kk) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      if (!live[i][0] && !live[i][1]) continue;
      const uint32_t lo[4] = {aa[i][0].x, aa[i][1].x, aa[i][0].y, aa[i][1].y};
      const uint32_t hi[4] = {aa[i][0].z, aa[i][1].z, aa[i][0].w, aa[i][1].w};
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < tokens8) {
          Mma<T>::run(acc[i][j], lo, xa[j].x, xa[j].y);
          Mma<T>::run(acc[i][j], hi, xa[j].z, xa[j].w);
        }
    }
  }
  float* mine_part = part + warp * (RT * 16 * kPitch);
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < tokens8) {
        *reinterpret_cast<float2*>(mine_part + (i * 16 + g) * kPitch + j * 8 + 2 * t) = make_float2(acc[i][j][0], acc[i][j][1]);
        *reinterpret_cast<float2*>(mine_part + (i * 16 + g + 8) * kPitch + j * 8 + 2 * t) = make_float2(acc[i][j][2], acc[i][j][3]);
      }
  __syncthreads();
  float* vp = v + ((long)blockIdx.z * rows + tile.start) * R + r0;
  for (int i = tid; i < tile.count * (RT * 16); i += 256) {
    const int token = i / (RT * 16), r = i % (RT * 16);
    if (r0 + r >= R) continue;
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) s += part[(w * RT * 16 + r) * kPitch + token];
    vp[(long)token * R + r] = s;
  }
}

// ---------------------------------------------------------------------------------------------
// out = y + scale * B v for a tile's rows and 512 columns of one slice, 64 a warp.  Output columns are the 16 rows of an MMA, tokens its
// columns; row g of product i of four stands for column 8 g + 2 i, row g + 8 for the next one, so that a thread ends with eight
// neighbouring columns of two tokens: one 16-byte access of y each (two in float32), a warp's accesses whole 128-byte lines.
// v is a float32 sum and stays one: it goes into the product as two 16-bit numbers whose sum carries 16 bits of it or more (22 in
// fp16), each row of it multiplied by a power of two that keeps it in fp16's range.
template <typename T, typename Y, int KT, bool ONE>
__global__ void __launch_bounds__(256, 1)
adapter_expand_kernel(const Y* y, long ldy, Y* out, long ldo, const T* b, const int* rank, const float* scale, const int* order,
                      const Tile* tiles, const float* v, int rows, int R, int rp, int planes, const Slices slices) {
  extern __shared__ char raw[];
  const int pitch = (rp + 15) / 16 * 16 + 8;              // 16-bit numbers of a token; rows 16 bytes apart in the banks
  T* hi = reinterpret_cast<T*>(raw);                      // [64][pitch]
  T* lo = hi + kTile * pitch;
  __shared__ float up[kTile];                             // a token's power of two, undone
  __shared__ int row_of[kTile];
  allow_dependents();
  dependency_wait();
  const Tile tile = tiles[blockIdx.x];
  if (tile.count == 0) return;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  int s = 0;
#pragma unroll
  for (int i = 1; i < kMaxSlices; ++i)
    if (i < slices.n && (int)blockIdx.y >= slices.block[i]) s = i;
  int c0 = 0, c1 = 0, b0 = 0;
#pragma unroll
  for (int i = 0; i < kMaxSlices; ++i)
    if (i == s) c0 = slices.start[i], c1 = slices.start[i + 1], b0 = slices.block[i];
  const int col = c0 + ((int)blockIdx.y - b0) * 512 + warp * 64 + g * 8;   // this thread's eight columns
  const bool in = col < c1;                                                // (slices are multiples of eight columns)
  if (tid < kTile) row_of[tid] = order[tile.start + min(tid, tile.count - 1)];
  const int mine = tile.slot < 0 ? 0 : rank[tile.slot * slices.n + s];
  if (mine == 0 && y == out) return;
  const float times = tile.slot < 0 ? 0.f : scale[tile.slot];
  const int steps = (mine + 15) / 16;
  if (mine > 0) {
    // four threads a token
    const int token = tid >> 2, q = tid & 3;
    const float* vr = v + ((long)tile.start + token) * R + s * rp;
    constexpr int NF = (ONE ? KT : kMaxRank / 16) * 4;
    float f[NF];
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < NF / 4; ++i) {
      const int j = i * 16 + q * 4;
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
      if (token < tile.count && j < mine) {   // (rp % 8 == 0: a group of four that starts inside the rank ends inside rp)
        for (int p = 0; p < planes; ++p) {
          const uint4 w = ld_stream_v4(vr + (long)p * rows * R + j);
          sum.x += __uint_as_float(w.x), sum.y += __uint_as_float(w.y);
          sum.z += __uint_as_float(w.z), sum.w += __uint_as_float(w.w);
        }
      }
      f[4 * i] = sum.x;
      f[4 * i + 1] = j + 1 < mine ? sum.y : 0.f;   // ranks past the slot's own are none, whatever the row holds
      f[4 * i + 2] = j + 2 < mine ? sum.z : 0.f;
      f[4 * i + 3] = j + 3 < mine ? sum.w : 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(f[4 * i + e]));
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // the largest magnitude goes to 2^13 .. 2^14 (2^100 and 2^-100 at most: beyond that it is 0 or no number for fp16 either way)
    const int e = top > 0.f && top < 3.4e38f ? max(-100, min(100, 13 - (int)((__float_as_uint(top) >> 23) & 0xffu) + 127)) : 0;
    const float down = __uint_as_float((uint32_t)(127 + e) << 23);
    if (q == 0) up[token] = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
    for (int i = 0; i < NF / 4; ++i) {
      const int j = i * 16 + q * 4;
      if (i < steps) {
        T h4[4], l4[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float w = f[4 * i + k] * down;
          h4[k] = narrow<T>(w);
          const float rest = w - to_f32<T>(h4[k]);
          l4[k] = narrow<T>(fabsf(w) < 3.4e38f ? rest : 0.f);
        }
        *reinterpret_cast<uint2*>(hi + token * pitch + j) = *reinterpret_cast<uint2*>(h4);
        *reinterpret_cast<uint2*>(lo + token * pitch + j) = *reinterpret_cast<uint2*>(l4);
      }
    }
  }
  __syncthreads();
  const int passes = ONE ? 1 : (steps + KT - 1) / KT;
  const T* bl = b + ((long)max(tile.slot, 0) * slices.start[slices.n] + col) * rp + 4 * t;
  uint32_t w[4][KT][4];
  auto fetch = [&](int pass) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int k = 0; k < KT; ++k) {
        const int step = pass * KT + k;
        const bool on = in && step < steps && step * 16 + 4 * t < rp;
        const uint2 p0 = on ? ld_v2(bl + (2 * i) * rp + step * 16) : make_uint2(0u, 0u);
        const uint2 p1 = on ? ld_v2(bl + (2 * i + 1) * rp + step * 16) : make_uint2(0u, 0u);
        w[i][k][0] = p0.x, w[i][k][2] = p0.y, w[i][k][1] = p1.x, w[i][k][3] = p1.y;
      }
  };
  if (ONE) fetch(0);
  constexpr int YV = sizeof(Y) / 2;   // 16-byte pieces of eight columns
#pragma unroll 1
  for (int half = 0; half < 2; ++half) {
    const int token0 = half * 32;
    if (token0 >= tile.count) break;
    uint4 old[4][2][YV];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int token = token0 + j * 8 + 2 * t + e;
#pragma unroll
        for (int p = 0; p < YV; ++p)
          if (in && token < tile.count) old[j][e][p] = ld_stream_v4(y + (long)row_of[token] * ldy + col + p * 4);
      }
    float acc[4][4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[j][i][0] = acc[j][i][1] = acc[j][i][2] = acc[j][i][3] = 0.f;
    for (int pass = 0; pass < passes; ++pass) {
      if (!ONE) fetch(pass);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (token0 + j * 8 >= tile.count) break;
#pragma unroll
        for (int k = 0; k < KT; ++k) {
          const int step = pass * KT + k;
          if (step >= steps) break;
          const int at = (token0 + j * 8 + g) * pitch + step * 16 + 4 * t;
          const uint2 h = *reinterpret_cast<const uint2*>(hi + at), l = *reinterpret_cast<const uint2*>(lo + at);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            Mma<T>::run(acc[j][i], w[i][k], l.x, l.y);
            Mma<T>::run(acc[j][i], w[i][k], h.x, h.y);
          }
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int token = token0 + j * 8 + 2 * t + e;
        if (!in || token >= tile.count) continue;
        if (mine > 0) {
          const float undo = up[token];
          Y* old8 = reinterpret_cast<Y*>(old[j][e]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            old8[2 * i] = narrow<Y>(__fmaf_rn(times, acc[j][i][e] * undo, to_f32<Y>(old8[2 * i])));
            old8[2 * i + 1] = narrow<Y>(__fmaf_rn(times, acc[j][i][2 + e] * undo, to_f32<Y>(old8[2 * i + 1])));
          }
        }
#pragma unroll
        for (int p = 0; p < YV; ++p)
          *reinterpret_cast<uint4*>(out + (long)row_of[token] * ldo + col + p * 4) = old[j][e][p];
      }
  }
}

// ---------------------------------------------------------------------------------------------
struct Plan {
  int R, rp, max_tiles, planes, k_range;
  size_t order_at, tiles_at, bytes;   // v lies at the scratch's start
};

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// Sizes in range: 0, or LQ_ERR_*.
int make_plan(int T, int K, int L, int rank, int S, Plan* p) {
  if (T <= 0 || K <= 0 || L <= 0 || rank <= 0 || S <= 0) return LQ_ERR_BAD_ARG;
  if (S > kMaxSlices || L > kMaxSlots || rank > kMaxRank || rank % 8 || K % 8 || T > (1 << 24) || K > (1 << 20))
    return LQ_ERR_SHAPE;
  p->rp = rank;
  p->R = S * rank;
  const int full = T / kTile, most = full + (T < L + 1 ? T : L + 1);
  p->max_tiles = most;
  // ranges of K: about two CTAs for every SM if tiles were full, at least 256 k each (a chunk of 32 for every warp)
  const int tiles = (T + kTile - 1) / kTile, chunks = (p->R + 63) / 64;
  int planes = 2 * sm_count() / (tiles * chunks);
  planes = planes < 1 ? 1 : planes > kMaxSplits ? kMaxSplits : planes;
  const int longest = (K + 255) / 256;
  if (planes > longest) planes = longest;
  p->k_range = ((K + planes - 1) / planes + 255) / 256 * 256;
  p->planes = (K + p->k_range - 1) / p->k_range;
  size_t at = up256((size_t)p->planes * T * p->R * sizeof(float));
  p->order_at = at;
  at += up256((size_t)T * sizeof(int));
  p->tiles_at = at;
  at += up256((size_t)p->max_tiles * sizeof(Tile));
  p->bytes = at;
  return LQ_OK;
}

template <typename F>
cudaError_t allow_smem(F* kernel, size_t bytes) {
  return bytes > 48 * 1024 ? cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) : cudaSuccess;
}

template <typename T, int RT>
cudaError_t launch_shrink(const Plan& p, const T* x, long ldx, const T* a, const int* rank, const int* order, const Tile* tiles,
                          float* v, int rows, int K, cudaStream_t st) {
  const size_t smem = (size_t)8 * RT * 16 * 66 * sizeof(float);
  cudaError_t e = allow_smem(adapter_shrink_kernel<T, RT>, smem);
  if (e != cudaSuccess) return e;
  return launch_overlapped(adapter_shrink_kernel<T, RT>, dim3(p.max_tiles, (p.R + RT * 16 - 1) / (RT * 16), p.planes), dim3(256),
                           smem, st, x, ldx, a, rank, order, tiles, v, rows, K, p.R, p.rp, p.k_range);
}

template <typename T, typename Y, int KT, bool ONE>
cudaError_t launch_expand(const Plan& p, const Y* y, long ldy, Y* out, long ldo, const T* b, const int* rank, const float* scale,
                          const int* order, const Tile* tiles, const float* v, int rows, const Slices& slices, cudaStream_t st) {
  const size_t smem = (size_t)2 * kTile * ((p.rp + 15) / 16 * 16 + 8) * sizeof(T);
  cudaError_t e = allow_smem(adapter_expand_kernel<T, Y, KT, ONE>, smem);
  if (e != cudaSuccess) return e;
  return launch_overlapped(adapter_expand_kernel<T, Y, KT, ONE>, dim3(p.max_tiles, slices.block[slices.n]), dim3(256), smem, st, y,
                           ldy, out, ldo, b, rank, scale, order, tiles, v, rows, p.R, p.rp, p.planes, slices);
}

template <typename T, typename Y>
cudaError_t run_expand(const Plan& p, const void* y, long ldy, void* out, long ldo, const void* b, const int* rank,
                       const float* scale, const int* order, const Tile* tiles, const float* v, int rows, const Slices& slices,
                       cudaStream_t st) {
  auto go = [&](auto launch) {
    return launch(p, static_cast<const Y*>(y), ldy, static_cast<Y*>(out), ldo, static_cast<const T*>(b), rank, scale, order, tiles, v,
                  rows, slices, st);
  };
  if (p.rp <= 16) return go(launch_expand<T, Y, 1, true>);
  if (p.rp <= 32) return go(launch_expand<T, Y, 2, true>);
  if (p.rp <= 64) return go(launch_expand<T, Y, 4, true>);
  return go(launch_expand<T, Y, 4, false>);
}

template <typename T>
cudaError_t run_add(const Plan& p, const void* x, long ldx, const void* a, const void* b, const int* rank, const float* scale,
                    const void* y, long ldy, int y_f32, void* out, long ldo, int rows, int K, const Slices& slices, int* order,
                    Tile* tiles, float* v, cudaStream_t st) {
  const T* xt = static_cast<const T*>(x);
  const T* at = static_cast<const T*>(a);
  cudaError_t e;
  if (p.R <= 16) e = launch_shrink<T, 1>(p, xt, ldx, at, rank, order, tiles, v, rows, K, st);
  else if (p.R <= 32) e = launch_shrink<T, 2>(p, xt, ldx, at, rank, order, tiles, v, rows, K, st);
  else e = launch_shrink<T, 4>(p, xt, ldx, at, rank, order, tiles, v, rows, K, st);
  if (e != cudaSuccess) return e;
  return y_f32 ? run_expand<T, float>(p, y, ldy, out, ldo, b, rank, scale, order, tiles, v, rows, slices, st)
               : run_expand<T, T>(p, y, ldy, out, ldo, b, rank, scale, order, tiles, v, rows, slices, st);
}

}  // namespace
}  // namespace lq

extern "C" size_t lq_adapters_scratch_bytes(int T, int K, int L, int rank, int n_slices) {
  lq::Plan p;
  return lq::make_plan(T, K, L, rank, n_slices, &p) == LQ_OK ? p.bytes : 0;
}

extern "C" int lq_adapters_add(const void* x, int dtype, long ldx, const void* a, const void* b, const int32_t* ranks,
                               const float* scales, const void* ids, int ids_64, const void* y, long ldy, int y_f32, void* out,
                               long ldo, int T, int K, int L, int rank, const int* widths, int n_slices, void* scratch,
                               size_t scratch_bytes, void* stream) {
  using namespace lq;
  if (!x || !a || !b || !ranks || !scales || !ids || !y || !out || !widths) return LQ_ERR_BAD_ARG;
  if (dtype != LQ_DT_BF16 && dtype != LQ_DT_F16) return LQ_ERR_BAD_ARG;
  Plan p;
  const int bad = make_plan(T, K, L, rank, n_slices, &p);
  if (bad) return bad;
  Slices slices = {};
  slices.n = n_slices;
  long N = 0;
  for (int s = 0; s < n_slices; ++s) {
    if (widths[s] <= 0) return LQ_ERR_BAD_ARG;
    if (widths[s] % 8 || widths[s] > (1 << 24)) return LQ_ERR_SHAPE;
    slices.start[s] = (int)N;
    N += widths[s];
    slices.block[s + 1] = slices.block[s] + (widths[s] + 511) / 512;
  }
  slices.start[n_slices] = (int)N;
  const int wide = y_f32 ? 4 : 2;
  auto odd = [](const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15) != 0; };
  if (odd(x) || odd(a) || odd(b) || odd(y) || odd(out) || ldx % 8 || ldx < 0 || (ldy * wide) % 16 || (ldo * wide) % 16 ||
      (T > 1 && (ldy < N || ldo < N)) || slices.block[n_slices] > 65535)
    return LQ_ERR_SHAPE;
  if (!scratch || odd(scratch) || scratch_bytes < p.bytes) return LQ_ERR_WORKSPACE;
  float* v = static_cast<float*>(scratch);
  int* order = reinterpret_cast<int*>(static_cast<char*>(scratch) + p.order_at);
  Tile* tiles = reinterpret_cast<Tile*>(static_cast<char*>(scratch) + p.tiles_at);
  cudaStream_t st = as_stream(stream);
  const size_t smem = (size_t)(3 * L + 5) * sizeof(int);
  cudaError_t e = allow_smem(adapter_plan_kernel, smem);
  if (e == cudaSuccess)
    e = launch_overlapped(adapter_plan_kernel, dim3(1), dim3(1024), smem, st, ids, ids_64 != 0, ranks, T, L, n_slices, y != out, order,
                          tiles, p.max_tiles);
  if (e == cudaSuccess)
    e = dtype == LQ_DT_BF16 ? run_add<__nv_bfloat16>(p, x, ldx, a, b, ranks, scales, y, ldy, y_f32, out, ldo, T, K, slices, order,
                                                     tiles, v, st)
                            : run_add<__half>(p, x, ldx, a, b, ranks, scales, y, ldy, y_f32, out, ldo, T, K, slices, order, tiles,
                                              v, st);
  if (e != cudaSuccess) {
    record_cuda_error(e, "adapters_add");
    return LQ_ERR_CUDA;
  }
  return check_launch("adapters_add");
}
