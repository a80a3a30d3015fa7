// Low-rank adapters of many requests at once, added to a projection's output:
//   v[t, s, j] = sum_k A[l, s, j, k] x[t, k]                                 l = ids[t], float32
//   out[t, n]  = (type of y)(y[t, n] + scale[l] * sum_j B[l, n, j] v[t, slice of n, j])
// A few rows: one kernel, a cluster of CTAs for up to eight rows of one adapter.  More: rows are put in the order of their adapters and
// cut into tiles of up to 64 rows of one adapter; a tile's rows times A (K cut over warps and CTAs); the result times B, added to y.
// The rows that a slot gets are known on the device only.
#include <type_traits>

#include "lq_common.cuh"
#include "lq_tc_ptx.cuh"

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
  int n, N, parts;             // all columns, all parts
  int start[kMaxSlices + 1];   // first column of a slice
  int part[kMaxSlices + 1];    // first part (the columns of a CTA, or of a warp) of a slice; parts end with their slice
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

// Two numbers rounded to a 16-bit type.
template <typename T> __device__ __forceinline__ uint32_t pack2(float2 v);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float2 v) {
  const __half2 h = __float22half2_rn(v);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float2 v) {
  const __nv_bfloat162 h = __float22bfloat162_rn(v);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T> __device__ __forceinline__ T narrow(float v);
template <> __device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// A coherent load that may stay in L1.
__device__ __forceinline__ uint2 ld_v2(const void* p) {
  uint2 r;
  asm volatile("ld.global.v2.u32 {%0,%1}, [%2];" : "=r"(r.x), "=r"(r.y) : "l"(p) : "memory");
  return r;
}

// The slot of a row, L where it has none.
__device__ __forceinline__ int slot_of(const void* ids, bool wide, long t, int L) {
  const long id = wide ? static_cast<const long long*>(ids)[t] : static_cast<const int*>(ids)[t];
  return id >= 0 && id < L ? (int)id : L;
}

// ---------------------------------------------------------------------------------------------
// Rows in the order of their slots, tiles.  One CTA.  The order within a slot hangs on atomics; no result does, since a row's sums
// are its own wherever it lies in a tile.
__global__ void __launch_bounds__(1024)
adapter_plan_kernel(const void* ids, bool wide, int T, int L, bool copy_rest, int* order, Tile* tiles,
                    int* done, int max_tiles) {
  extern __shared__ int counts[];
  int* first = counts;                // [L + 2] rows before a slot's
  int* tile0 = counts + L + 2;        // [L + 2] tiles before a slot's
  int* next = tile0 + L + 2;          // [L + 1] counts, then the next free place
  __shared__ int warp_sum[2][32];
  allow_dependents();
  dependency_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int i = tid; i <= L; i += blockDim.x) next[i] = 0;
  __syncthreads();
  constexpr int B = 8;   // ids of a thread that are on their way together
  int slot[B];
  auto take = [&](int t0) {
#pragma unroll
    for (int i = 0; i < B; ++i) {
      const int t = t0 + i * 1024 + tid;
      slot[i] = t < T ? slot_of(ids, wide, t, L) : -1;
    }
  };
  for (int t0 = 0; t0 < T; t0 += B * 1024) {
    take(t0);
#pragma unroll
    for (int i = 0; i < B; ++i) {
      if (t0 + i * 1024 >= T) break;
      const unsigned same = __match_any_sync(0xffffffffu, slot[i]);
      if (slot[i] >= 0 && lane == __ffs(same) - 1) atomicAdd(&next[slot[i]], __popc(same));
    }
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
    done[i] = 0;
  }
  for (int t0 = 0; t0 < T; t0 += B * 1024) {
    if (T > B * 1024) take(t0);
#pragma unroll
    for (int i = 0; i < B; ++i) {
      if (t0 + i * 1024 >= T) break;
      const unsigned same = __match_any_sync(0xffffffffu, slot[i]);
      const int leader = __ffs(same) - 1;
      int at = 0;
      if (slot[i] >= 0 && lane == leader) at = atomicAdd(&next[slot[i]], __popc(same));
      at = __shfl_sync(0xffffffffu, at, leader) + __popc(same & ((1u << lane) - 1));
      if (slot[i] >= 0) order[at] = t0 + i * 1024 + tid;
    }
  }
}

// ---------------------------------------------------------------------------------------------
// v = A x.  Ranks are the 16 rows of an MMA, eight tokens its columns, so that both operands come straight from their row-major
// matrices into registers.  The order of k within a product is free: thread t of a quad takes the eight neighbours
// 8 t .. 8 t + 7 of 32 k for both operands, one 16-byte load each.

// A float32 sum goes into the second product as two 16-bit numbers whose sum carries 16 bits of it or more (22 in fp16), multiplied by
// a power of two that keeps a row's sums of one slice in fp16's range.
struct Power {
  float down, up;
};
__device__ __forceinline__ Power power_of(float top) {   // of the largest magnitude: it goes to 2^13 .. 2^14
  const int e = top > 0.f && top < 3.4e38f ? max(-100, min(100, 140 - (int)((__float_as_uint(top) >> 23) & 0xffu))) : 0;
  return {__uint_as_float((uint32_t)(127 + e) << 23), __uint_as_float((uint32_t)(127 - e) << 23)};
}
template <typename T>
__device__ __forceinline__ void halves(float v, T& hi, T& lo) {
  hi = narrow<T>(v);
  lo = narrow<T>(fabsf(v) < 3.4e38f ? v - to_f32<T>(hi) : 0.f);
}

__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool on) {   // zeros where it is not on
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_but() {   // all copies but those of the last N groups are there
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void bulk_store(void* to, uint32_t from, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(to), "r"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void commit_stores() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void stores_read_but() {   // all bulk stores but those of the last N groups have read shared memory
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}
constexpr uint64_t kWaitLimit = 2000000000ull;
__device__ __forceinline__ bool await(uint32_t bar, uint32_t parity, int* status, int site) {
  const bool ok = ptx::mbar_wait_bounded(bar, parity, kWaitLimit);
  if (!ok) atomicExch(status, site);
  return ok;
}
__device__ __forceinline__ uint4 lds_v4(uint32_t at) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(at) : "memory");
  return r;
}

// A tile's rows, 16 RT ranks and one range of K.  Sixteen warps take turns at the 32-k chunks of the range, each thread's pieces on their
// way into places of its own in shared memory a chunk ahead (nobody else reads them: no barrier).  The warps' sums meet in shared memory
// and go to plane blockIdx.z of v [planes][T][R] (R = slices x stack rank), in the order of the plan; the last CTA of a tile adds up the
// planes, in their order, and writes the sums' halves, vv [slices][T][stack rank / 4][2][4], and the power of two of each.
// Bound by the stream of x and its latencies: 8192 rows of 14336 at rank 16 57 us (235 MB, 4.1 TB/s); eight warps 74, rows by bulk
// copies of 512 bytes 150.
constexpr int kShrinkThreads = 512;
template <int RT>
struct Shrink {
  static constexpr int kPieces = 8 + 2 * RT, kStage = kPieces * kShrinkThreads * 16, kStages = 2;
  static constexpr int kSums = kShrinkThreads / 32 * RT * 16 * 66 * (int)sizeof(float);
  static constexpr int kBytes = kStage * kStages > kSums ? kStage * kStages : kSums;
};

template <typename T, int RT>
__global__ void __launch_bounds__(kShrinkThreads, 1)
adapter_shrink_kernel(const T* x, long ldx, const T* a, const int* rank, const int* order, const Tile* tiles, int* done, float* v,
                      T* vv, float* up, int rows, int K, int R, int rp, int k_range) {
  extern __shared__ __align__(128) char smem[];   // [stages][pieces][threads] of 16 bytes; then float [warps][RT * 16][66]
  __shared__ int row_of[kTile];
  __shared__ bool last;
  constexpr int kPitch = 66, STAGES = Shrink<RT>::kStages, WARPS = kShrinkThreads / 32, kPiece = kShrinkThreads * 16;
  allow_dependents();
  dependency_wait();
  const Tile tile = tiles[blockIdx.x];
  if (tile.count == 0 || tile.slot < 0) return;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  if (tid < kTile) row_of[tid] = order[tile.start + min(tid, tile.count - 1)];
  const int r0 = blockIdx.y * (RT * 16), S = R / rp;
  const int k0 = blockIdx.z * k_range;
  int k1 = k0;        // (nothing to sum where no rank is reached)
  bool live[RT][2];   // the eight-row halves of the rank tiles that the slices' ranks reach (rp % 8 == 0)
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = r0 + i * 16 + h * 8;
      live[i][h] = r < R && r % rp < rank[tile.slot * S + r / rp];
      if (live[i][h]) k1 = min(K, k0 + k_range);
    }
  const int tokens8 = (tile.count + 7) / 8;
  float acc[RT][8][4];
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[i][j][0] = acc[i][j][1] = acc[i][j][2] = acc[i][j][3] = 0.f;
  __syncthreads();
  const int first = k0 + warp * 32;
  // (volatile products: a thread's next copies into a place are behind those that used what it held)
  const T* xr[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) xr[j] = x + (long)row_of[j * 8 + g] * ldx + 8 * t;
  const T* ar = a + ((long)tile.slot * R + r0 + g) * K + 8 * t;
  const uint32_t places = smem_u32(smem) + tid * 16;
  auto ask = [&](int k, int stage) {
    if (k < k1) {
      const bool in = k + 8 * t < k1;
      const uint32_t to = places + stage * Shrink<RT>::kStage;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < tokens8) copy16(to + j * kPiece, in ? xr[j] + k : x, in);
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (live[i][h]) copy16(to + (8 + 2 * i + h) * kPiece, in ? ar + (long)(i * 16 + h * 8) * K + k : a, in);
    }
    commit_copies();
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) ask(first + i * (32 * WARPS), i);
  int stage = 0;
  for (int k = first; k < k1; k += 32 * WARPS) {
    copies_but<STAGES - 2>();
    const uint32_t from = places + stage * Shrink<RT>::kStage;
    ask(k + (STAGES - 1) * (32 * WARPS), stage == 0 ? STAGES - 1 : stage - 1);   // (where this thread read the chunk before)
    stage = stage == STAGES - 1 ? 0 : stage + 1;
    uint4 aa[RT][2];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) aa[i][h] = live[i][h] ? lds_v4(from + (8 + 2 * i + h) * kPiece) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (j >= tokens8) break;
      const uint4 xa = lds_v4(from + j * kPiece);
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        const uint32_t lo[4] = {aa[i][0].x, aa[i][1].x, aa[i][0].y, aa[i][1].y};
        const uint32_t hi[4] = {aa[i][0].z, aa[i][1].z, aa[i][0].w, aa[i][1].w};
        Mma<T>::run(acc[i][j], lo, xa.x, xa.y);
        Mma<T>::run(acc[i][j], hi, xa.z, xa.w);
      }
    }
  }
  copies_but<0>();
  __syncthreads();   // every place has been read: they take the sums
  float* part = reinterpret_cast<float*>(smem);
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
  for (int i = tid; i < tile.count * (RT * 16); i += kShrinkThreads) {
    const int token = i / (RT * 16), r = i % (RT * 16);
    if (r0 + r >= R) continue;
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) s += part[(w * RT * 16 + r) * kPitch + token];
    vp[(long)token * R + r] = s;
  }
  __threadfence();
  __syncthreads();
  if (tid == 0) last = atomicAdd(done + blockIdx.x, 1) == (int)(gridDim.y * gridDim.z) - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  // a row's sums of one slice: four threads, four neighbouring ranks of 16 each, four planes on their way at a time
  for (int item = tid >> 2; item - (tid >> 2) < tile.count * S; item += kShrinkThreads / 4) {
    const int q = tid & 3, token = min(item, tile.count * S - 1) / S, s = min(item, tile.count * S - 1) % S;
    const long row = (long)tile.start + token;
    const int mine = min(rank[tile.slot * S + s], rp), planes = gridDim.z;
    const float* from = v + row * R + s * rp + q * 4;
    const long plane = (long)rows * R;
    auto sum4 = [&](int j) {   // (ranks past the slice's own are none, whatever the row holds)
      float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
      if (j + q * 4 < mine)
        for (int p = 0; p < planes; p += 4) {
          uint4 w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = p + e < planes ? __ldcg(reinterpret_cast<const uint4*>(from + (p + e) * plane + j)) : make_uint4(0, 0, 0, 0);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            f.x += __uint_as_float(w[e].x), f.y += __uint_as_float(w[e].y);
            f.z += __uint_as_float(w[e].z), f.w += __uint_as_float(w[e].w);
          }
        }
      const int j0 = j + q * 4;
      return make_float4(f.x, j0 + 1 < mine ? f.y : 0.f, j0 + 2 < mine ? f.z : 0.f, j0 + 3 < mine ? f.w : 0.f);
    };
    float4 keep[4];   // the first 64 ranks stay in registers
    float top = 0.f;
    auto take = [&](const float4& f) {
      top = fmaxf(top, fmaxf(fmaxf(fabsf(f.x), fabsf(f.y)), fmaxf(fabsf(f.z), fabsf(f.w))));
    };
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      keep[i] = sum4(i * 16);
      take(keep[i]);
    }
    for (int j = 64; j < mine; j += 16) take(sum4(j));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const Power power = power_of(top);
    if (item >= tile.count * S) continue;
    if (q == 0) up[(long)s * rows + row] = power.up;
    T* to = vv + (((long)s * rows + row) * rp + q * 4) * 2;
    auto write = [&](int j, const float4& f) {
      if (j + q * 4 >= rp) return;
      __align__(16) T e[8];   // the first halves of four ranks, then the second
      halves<T>(f.x * power.down, e[0], e[4]);
      halves<T>(f.y * power.down, e[1], e[5]);
      halves<T>(f.z * power.down, e[2], e[6]);
      halves<T>(f.w * power.down, e[3], e[7]);
      *reinterpret_cast<uint4*>(to + j * 2) = *reinterpret_cast<uint4*>(e);
    };
#pragma unroll
    for (int i = 0; i < 4; ++i) write(i * 16, keep[i]);
    for (int j = 64; j < rp; j += 16) write(j, sum4(j));
  }
}

// ---------------------------------------------------------------------------------------------
// out = y + scale * B v.  Output columns are the 16 rows of an MMA, eight tokens its columns; row g of product i of MT stands for column
// 2 MT g + 2 i of a warp's 16 MT, row g + 8 for the next one, so that a thread ends with 2 MT neighbouring columns of two tokens: whole
// 16-byte accesses of y (8 with MT = 2), a warp's in whole lines.

// This thread's part of 16 MT columns of B (`b`: its own first), KT * 16 ranks of the `left` that their rows still hold.
template <int KT, int MT>
__device__ __forceinline__ void fetch_columns(uint32_t (&w)[MT][KT][4], const void* b, bool in, int steps, int rp, int left, int t) {
  const char* p = static_cast<const char*>(b) + 8 * t;
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int k = 0; k < KT; ++k) {
      const bool on = in && k < steps && k * 16 + 4 * t < left;
      const uint2 p0 = on ? ld_v2(p + (2 * i) * rp * 2 + k * 32) : make_uint2(0u, 0u);
      const uint2 p1 = on ? ld_v2(p + (2 * i + 1) * rp * 2 + k * 32) : make_uint2(0u, 0u);
      w[i][k][0] = p0.x, w[i][k][2] = p0.y, w[i][k][1] = p1.x, w[i][k][3] = p1.y;
    }
}

// Which slice a part of `columns` columns belongs to, its first column and the slice's end.
struct Where {
  int s, col, end;
};
__device__ __forceinline__ Where where_is(const Slices& slices, int part, int columns) {
  int s = 0, start = slices.start[0], end = slices.start[1], first = 0;
#pragma unroll
  for (int i = 1; i < kMaxSlices; ++i)
    if (i < slices.n && part >= slices.part[i]) s = i, start = slices.start[i], end = slices.start[i + 1], first = slices.part[i];
  return {s, start + (part - first) * columns, end};
}

// A CTA has 128 MT columns of one slice, 16 MT a warp, and walks over a range of tiles, up to 16 rows at a time; B's part stays in
// registers as long as the slot does.  Rows of y come by bulk copies, two a warp, with their halves of v, and results go back the same
// way; what lies between is shared memory and MMAs.  The copies alone take 23 us for 8192 rows of 4096 and 178 for 28672 (floors 21 and
// 144); with the products (rank 16, and 64) it is 32 and 365: issue of instructions and copies.  All copying by one warp: 39 and 438.
constexpr int kPart = 16;
template <typename Y, int KT, int MT>
struct Expand {
  static constexpr int kRowY = 128 * MT * (int)sizeof(Y) + 16;   // (16 apart in the banks: a quad's rows without conflicts)
  static constexpr int kV = kPart * KT * 64, kUp = 128, kStage = kPart * kRowY + kV + kUp;
  static constexpr int kFit = (KT <= 1 ? 72 : KT <= 4 ? 108 : 216) * 1024 / kStage, kStages = kFit < 2 ? 2 : kFit > 4 ? 4 : kFit;
};

template <typename T, typename Y, int KT, int MT>
__global__ void __launch_bounds__(256, KT <= 1 ? 3 : KT <= 4 ? 2 : 1)
adapter_expand_kernel(const Y* y, long ldy, Y* out, long ldo, const T* b, const int* rank, const float* scale, const int* order,
                      const Tile* tiles, const T* vv, const float* up, int rows, int rp, int max_tiles, int tiles_each,
                      const Slices slices, int* status) {
  extern __shared__ __align__(128) char smem[];   // stages of: y [kPart][kRowY], v [kPart][rp / 4][2][4], powers [kPart]
  using E = Expand<Y, KT, MT>;
  constexpr int COLS = 2 * MT, STAGES = E::kStages, BYTES = COLS * (int)sizeof(Y), PB = BYTES < 16 ? BYTES : 16, PIECES = BYTES / PB;
  __shared__ __align__(8) uint64_t bars[STAGES];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const uint32_t full = smem_u32(bars), ring = smem_u32(smem);
  if (tid == 0) {
#pragma unroll
    for (int i = 0; i < STAGES; ++i) ptx::mbar_init(full + 8 * i, kPart);
    ptx::fence_mbar_init();
  }
  allow_dependents();
  dependency_wait();
  __syncthreads();
  const Where at = where_is(slices, blockIdx.x, 128 * MT);
  const int tile0 = (int)blockIdx.y * tiles_each, tile_end = min(max_tiles, tile0 + tiles_each);
  const Tile none = {-1, 0, 0, 0};
  const bool in_place = y == out;
  auto tile_at = [&](int i) { return i < tile_end ? tiles[i] : none; };
  auto rank_at = [&](const Tile& tile) { return tile.slot < 0 ? 0 : min(rank[tile.slot * slices.n + at.s], rp); };

  // What the first two lanes of a warp ask for: row 2 warp + lane of part `ap` of tile `asked`, the row's index and power known a part ahead.
  const bool copies = lane < kPart / 8;
  const int mine_token = warp * (kPart / 8) + lane;
  const uint32_t row_bytes = min(128 * MT, at.end - at.col) * (int)sizeof(Y);
  int ai = tile0, ap = 0, arow = 0;
  float apower = 0.f;
  Tile asked = tile_at(ai);
  int arank = rank_at(asked);
  auto look = [&]() {
    if (copies && ap * kPart + mine_token < asked.count) {
      arow = order[asked.start + ap * kPart + mine_token];
      if (arank > 0) apower = up[(long)at.s * rows + asked.start + ap * kPart + mine_token];
    }
  };
  look();
  auto ask = [&](int stage) {   // the row that this lane will write back from there, -1: none
    int held = -1;
    if (asked.count == 0) return held;
    if (copies) {
      const uint32_t to = ring + stage * E::kStage, bar = full + 8 * stage;
      const int left = min(kPart, asked.count - ap * kPart);
      const bool on = mine_token < left && !(in_place && arank == 0), first = tid == 0 && arank > 0;
      if (on) held = arow;
      if (arank > 0 && mine_token < left)
        asm volatile("st.shared.f32 [%0], %1;" ::"r"(to + kPart * E::kRowY + E::kV + mine_token * 4), "f"(apower) : "memory");
      ptx::mbar_expect_tx(bar, (on ? row_bytes : 0) + (first ? left * rp * 4 : 0));
      if (on) ptx::bulk_load(to + mine_token * E::kRowY, y + (long)arow * ldy + at.col, row_bytes, bar);
      if (first)
        ptx::bulk_load(to + kPart * E::kRowY, vv + ((long)at.s * rows + asked.start + ap * kPart) * rp * 2, left * rp * 4, bar);
    }
    if (++ap * kPart >= asked.count) {
      ap = 0;
      asked = tile_at(++ai);
      arank = rank_at(asked);
    }
    look();
    return held;
  };
  int held[STAGES];   // by parts, the one in hand first
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) held[i] = ask(i);

  const int col = at.col + warp * (16 * MT) + g * COLS;
  const bool in = col < at.end;
  int turn = 0, stage = 0, slot = -2, mine = 0, steps = 0;
  float times = 0.f;
  bool lost = false;
  uint32_t w[MT][KT][4];
  Tile tile = tile_at(tile0);
  for (int i = tile0; tile.count > 0; ++i) {
    const Tile after = tile_at(i + 1);
    if (tile.slot != slot) {
      slot = tile.slot;
      mine = rank_at(tile);
      times = slot < 0 ? 0.f : scale[slot];
      steps = (mine + 15) / 16;
      fetch_columns<KT, MT>(w, b + ((long)max(slot, 0) * slices.N + col) * rp, in, steps, rp, rp, t);
    }
    for (int part = 0; part * kPart < tile.count; ++part, ++turn) {
      const int left = min(kPart, tile.count - part * kPart);
      if (!lost) lost = !await(full + 8 * stage, (turn / STAGES) & 1, status, 181);   // (reported: no more waiting, wrong rows)
      const uint32_t from = ring + stage * E::kStage, fv = from + kPart * E::kRowY;
      if (mine > 0 && warp * (16 * MT) < at.end - at.col) {
#pragma unroll
        for (int j = 0; j < kPart / 8; ++j) {
          if (j * 8 >= left) break;
          float acc[MT][4];
#pragma unroll
          for (int m = 0; m < MT; ++m) acc[m][0] = acc[m][1] = acc[m][2] = acc[m][3] = 0.f;
          const uint32_t va = fv + (min(j * 8 + g, left - 1) * rp + 4 * t) * 4;
          constexpr int V = KT < 4 ? KT : 4;   // steps whose halves are read ahead of their products
#pragma unroll
          for (int k0 = 0; k0 < KT; k0 += V) {
            uint4 v[V];
#pragma unroll
            for (int k = 0; k < V; ++k)
              v[k] = k0 + k < steps && (k0 + k) * 16 + 4 * t < rp ? lds_v4(va + (k0 + k) * 64) : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int k = 0; k < V; ++k) {
              if (k0 + k >= steps) break;
#pragma unroll
              for (int m = 0; m < MT; ++m) Mma<T>::run(acc[m], w[m][k0 + k], v[k].z, v[k].w);
#pragma unroll
              for (int m = 0; m < MT; ++m) Mma<T>::run(acc[m], w[m][k0 + k], v[k].x, v[k].y);
            }
          }
          float undo[2];
          asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(undo[0]), "=f"(undo[1]) : "r"(fv + E::kV + (j * 8 + 2 * t) * 4) : "memory");
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int token = j * 8 + 2 * t + e;
            if (!in || token >= left) continue;
            const uint32_t piece = from + token * E::kRowY + (warp * (16 * MT) + g * COLS) * (int)sizeof(Y);
#pragma unroll
            for (int p = 0; p < PIECES; ++p) {
              constexpr int EACH = PB / (int)sizeof(Y);   // columns of a piece
              uint32_t o[4];
              if constexpr (PB == 16) {
                const uint4 q = lds_v4(piece + p * 16);
                o[0] = q.x, o[1] = q.y, o[2] = q.z, o[3] = q.w;
              } else {
                asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(o[0]), "=r"(o[1]) : "r"(piece) : "memory");
              }
#pragma unroll
              for (int c = 0; c < EACH; c += 2) {
                const int m = (p * EACH + c) / 2;   // the MMA row pair of columns c and c + 1
                const float f0 = acc[m][e] * undo[e], f1 = acc[m][2 + e] * undo[e];
                if constexpr (sizeof(Y) == 2) {
                  const float2 old = unpack2<Y>(o[c / 2]);
                  o[c / 2] = pack2<Y>(make_float2(__fmaf_rn(times, f0, old.x), __fmaf_rn(times, f1, old.y)));
                } else {
                  o[c] = __float_as_uint(__fmaf_rn(times, f0, __uint_as_float(o[c])));
                  o[c + 1] = __float_as_uint(__fmaf_rn(times, f1, __uint_as_float(o[c + 1])));
                }
              }
              if constexpr (PB == 16)
                asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(piece + p * 16), "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3]) : "memory");
              else
                asm volatile("st.shared.v2.u32 [%0], {%1,%2};" ::"r"(piece), "r"(o[0]), "r"(o[1]) : "memory");
            }
          }
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // what this thread wrote and read, ahead of the bulk copies
      __syncthreads();
      if (held[0] >= 0) bulk_store(out + (long)held[0] * ldo + at.col, from + mine_token * E::kRowY, row_bytes);
      commit_stores();
#pragma unroll
      for (int h = 0; h + 2 < STAGES; ++h) held[h] = held[h + 1];
      stores_read_but<1>();   // the part before this one has left its stage
      held[STAGES - 2] = ask(stage == 0 ? STAGES - 1 : stage - 1);
      stage = stage == STAGES - 1 ? 0 : stage + 1;
    }
    tile = after;
  }
  if (lost)   // what may still be on its way ends before the CTA does
    for (int i = 1; i <= STAGES; ++i)
      if (turn >= i) ptx::mbar_wait_bounded(full + 8 * ((turn - i) % STAGES), ((turn - i) / STAGES) & 1, kWaitLimit);
  stores_read_but<0>();
}

// ---------------------------------------------------------------------------------------------
// A few rows, in one launch.  A cluster for up to eight rows of one adapter (the cluster of the first of them; the others' end at
// once): its CTAs share out K for the first product, exchange their sums through distributed shared memory, and share out
// the columns for the second.  A's and B's rows are read from memory straight into MMA operands, B's lines asked for into L2 at the start.
// Bound by the chain of latencies (ids, rows and weights, the exchange, y): 6.2 us for one row of 4096 to 4096, 16 for 32 rows with adapters of
// their own to 6144 (three launches: 12 and 26).
constexpr int kFewRanks = 512;    // slices x stack rank

__device__ __forceinline__ float4 peer_v4(uint32_t at, int cta) {
  uint32_t there;
  float4 f;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(at), "r"(cta));
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(f.x), "=f"(f.y), "=f"(f.z), "=f"(f.w) : "r"(there) : "memory");
  return f;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// RT tiles of 16 ranks at a time in the first product, KT steps of 16 in the second.  The code is kept short: a launch that
// takes a few us waits for its instructions as well (four groups of columns unrolled: one token 9.6 us instead of 7.5).
template <typename T, typename Y, int RT, int KT>
__global__ void __launch_bounds__(256, 2)
adapter_few_kernel(const T* x, long ldx, const Y* y, long ldy, Y* out, long ldo, const T* a, const T* b, const int* rank,
                   const float* scale, const void* ids, bool wide, int rows, int K, int L, int R, int rp, const Slices slices) {
  extern __shared__ __align__(128) char smem[];
  float* mine_v = reinterpret_cast<float*>(smem);               // [R][8] this CTA's sums, which its peers read
  float* all_v = mine_v + R * 8;                                // [R][8]
  float* part_v = all_v + R * 8;                                  // [8 warps][16 RT][8]; then the halves: [8 tokens][R / 4 + 1] of 16 bytes
  __shared__ unsigned same_of[8];
  __shared__ int row_of[8];
  __shared__ float up_of[8][kMaxSlices];
  __shared__ int rank_of[kMaxSlices];
  allow_dependents();
  dependency_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int cta = blockIdx.x, ctas = gridDim.x, m = blockIdx.y, S = slices.n, N = slices.N;
  const int slot = slot_of(ids, wide, m, L);
  const bool in_place = y == out;
  if (slot == L) {
    if (!in_place) {
      constexpr int EACH = 16 / (int)sizeof(Y);
      for (int n = (cta * 256 + tid) * EACH; n < N; n += ctas * 256 * EACH)
        *reinterpret_cast<uint4*>(out + m * ldo + n) = ld_stream_v4(y + m * ldy + n);
    }
    return;
  }
  const float times = scale[slot];
  if (tid < S) rank_of[tid] = min(rank[slot * S + tid], rp);
  const bool like = tid < rows && slot_of(ids, wide, tid, L) == slot;
  const unsigned same = __ballot_sync(0xffffffffu, like);
  if (lane == 0) same_of[warp] = same;
  __syncthreads();
  int before = 0, ahead = 0, total = 0;   // rows of the slot ahead of this thread's, of this cluster's, and all
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    const unsigned s = same_of[w];
    total += __popc(s);
    before += w < warp ? __popc(s) : w == warp ? __popc(s & ((1u << lane) - 1)) : 0;
    ahead += w < m / 32 ? __popc(s) : w == m / 32 ? __popc(s & ((1u << (m & 31)) - 1)) : 0;
  }
  if (ahead % 8) return;
  const int count = min(8, total - ahead);
  if (like && before >= ahead && before < ahead + 8) row_of[before - ahead] = tid;
  const T* al = a + (long)slot * R * K;
  const T* bl = b + (long)slot * N * rp;
  const int group0 = cta * 8 + warp, groups = ctas * 8;
  for (int i = group0; i < slices.parts; i += groups) {   // 64 rows of B are 64 rp neighbours
    const Where at = where_is(slices, i, 64);
    for (int line = lane; line < rp; line += 32)
      if (at.col + line * 64 / rp < at.end)
        asm volatile("prefetch.global.L2 [%0];" ::"l"(reinterpret_cast<const char*>(bl + (long)at.col * rp) + line * 128));
  }
  __syncthreads();
  const T* xr = x + (long)row_of[min(g, count - 1)] * ldx + 8 * t;
  const int chunks = (K + 31) / 32;
  for (int p = 0; p < R; p += 16 * RT) {
    float acc[RT][4];
    bool live[RT][2];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = p + i * 16 + h * 8;
        live[i][h] = r < R && r % rp < rank_of[min(r, R - 1) / rp];
      }
    }
    const T* ar = al + (long)(p + g) * K + 8 * t;
    for (int c = group0; c < chunks; c += 2 * groups) {   // two chunks of 32 k on their way
      uint4 xa[2], aa[2][RT][2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int k = (c + u * groups) * 32;
        const bool in = k + 8 * t < K;
        xa[u] = in ? ld_stream_v4(xr + k) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            aa[u][i][h] = in && live[i][h] ? ld_stream_v4(ar + (long)(i * 16 + h * 8) * K + k) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < RT; ++i) {
          const uint32_t lo[4] = {aa[u][i][0].x, aa[u][i][1].x, aa[u][i][0].y, aa[u][i][1].y};
          const uint32_t hi[4] = {aa[u][i][0].z, aa[u][i][1].z, aa[u][i][0].w, aa[u][i][1].w};
          Mma<T>::run(acc[i], lo, xa[u].x, xa[u].y);
          Mma<T>::run(acc[i], hi, xa[u].z, xa[u].w);
        }
    }
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<float2*>(part_v + (warp * (16 * RT) + i * 16 + h * 8 + g) * 8 + 2 * t) = make_float2(acc[i][2 * h], acc[i][2 * h + 1]);
    __syncthreads();
    for (int i = tid; i < min(16 * RT, R - p) * 8; i += 256) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) s += part_v[w * (128 * RT) + i];
      mine_v[p * 8 + i] = s;
    }
    __syncthreads();
  }
  cluster_arrive();
  cluster_wait();
  for (int i = tid; i < R * 2; i += 256) {
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c = 0; c < ctas; ++c) {
      const float4 f = peer_v4(smem_u32(mine_v) + i * 16, c);
      s.x += f.x, s.y += f.y, s.z += f.z, s.w += f.w;
    }
    reinterpret_cast<float4*>(all_v)[i] = s;
  }
  __syncthreads();
  cluster_arrive();   // (waited for at the end: peers may be reading this CTA's sums)
  T* halves_of = reinterpret_cast<T*>(part_v) + warp * (R / 4 + 1) * 8;   // a warp for a token
  for (int s = 0; s < S; ++s) {
    const int mine = rank_of[s];
    float top = 0.f;   // (ranks past the slice's own are none, whatever the row holds)
    for (int j = lane; j < mine; j += 32) top = fmaxf(top, fabsf(all_v[(s * rp + j) * 8 + warp]));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const Power power = power_of(top);
    if (lane == 0) up_of[warp][s] = power.up;
    for (int j = lane; j < rp; j += 32) {
      T h, l;
      halves<T>(j < mine ? all_v[(s * rp + j) * 8 + warp] * power.down : 0.f, h, l);
      T* to = halves_of + (s * rp + j) / 4 * 8 + j % 4;
      to[0] = h, to[4] = l;
    }
  }
  __syncthreads();
  constexpr int YV = sizeof(Y) / 2;   // 16-byte pieces of eight columns
  for (int i = group0; i < slices.parts; i += groups) {
    const Where at = where_is(slices, i, 64);
    const int mine = rank_of[at.s], steps = (mine + 15) / 16, col = at.col + g * 8;
    if (mine == 0 && in_place) continue;
    const bool in = col < at.end;
    uint4 old[2][YV];
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int p = 0; p < YV; ++p)
        if (in && 2 * t + e < count) old[e][p] = ld_stream_v4(y + row_of[2 * t + e] * ldy + col + p * 4);
    float acc[4][4];
#pragma unroll
    for (int q = 0; q < 4; ++q) acc[q][0] = acc[q][1] = acc[q][2] = acc[q][3] = 0.f;
    const uint32_t va = smem_u32(part_v) + (g * (R / 4 + 1) + (at.s * rp) / 4 + t) * 16;
    for (int k0 = 0; k0 < steps; k0 += KT) {
      uint32_t w[4][KT][4];
      fetch_columns<KT, 4>(w, bl + (long)col * rp + k0 * 16, in, steps - k0, rp, rp - k0 * 16, t);
#pragma unroll
      for (int k = 0; k < KT; ++k) {
        if (k0 + k >= steps) break;
        const uint4 v = (k0 + k) * 16 + 4 * t < rp ? lds_v4(va + (k0 + k) * 64) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int q = 0; q < 4; ++q) Mma<T>::run(acc[q], w[q][k], v.z, v.w);
#pragma unroll
        for (int q = 0; q < 4; ++q) Mma<T>::run(acc[q], w[q][k], v.x, v.y);
      }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      if (!in || 2 * t + e >= count) continue;
      if (mine > 0) {
        const float undo = up_of[2 * t + e][at.s];
        uint32_t* o = reinterpret_cast<uint32_t*>(old[e]);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float f0 = acc[q][e] * undo, f1 = acc[q][2 + e] * undo;
          if constexpr (sizeof(Y) == 2) {
            const float2 before = unpack2<Y>(o[q]);
            o[q] = pack2<Y>(make_float2(__fmaf_rn(times, f0, before.x), __fmaf_rn(times, f1, before.y)));
          } else {
            o[2 * q] = __float_as_uint(__fmaf_rn(times, f0, __uint_as_float(o[2 * q])));
            o[2 * q + 1] = __float_as_uint(__fmaf_rn(times, f1, __uint_as_float(o[2 * q + 1])));
          }
        }
      }
#pragma unroll
      for (int p = 0; p < YV; ++p) *reinterpret_cast<uint4*>(out + row_of[2 * t + e] * ldo + col + p * 4) = old[e][p];
    }
  }
  cluster_wait();
}

// ---------------------------------------------------------------------------------------------
struct Plan {
  int R, rp, max_tiles, planes, k_range;
  size_t vv_at, up_at, order_at, tiles_at, done_at, bytes;   // v lies at the scratch's start
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
  // ranges of K: about one CTA for every SM if tiles were full, at least 512 k each
  const int tiles = (T + kTile - 1) / kTile, chunks = (p->R + 31) / 32;
  int planes = sm_count() / (tiles * chunks);
  planes = planes < 1 ? 1 : planes > kMaxSplits ? kMaxSplits : planes;
  const int longest = (K + 511) / 512;
  if (planes > longest) planes = longest;
  p->k_range = ((K + planes - 1) / planes + 255) / 256 * 256;
  p->planes = (K + p->k_range - 1) / p->k_range;
  const size_t cells = (size_t)T * p->R;
  size_t at = up256(p->planes * cells * sizeof(float));
  p->vv_at = at, at += up256(cells * 4);
  p->up_at = at, at += up256((size_t)T * S * sizeof(float));
  p->order_at = at, at += up256((size_t)T * sizeof(int));
  p->tiles_at = at, at += up256((size_t)p->max_tiles * sizeof(Tile));
  p->done_at = at, at += up256((size_t)p->max_tiles * sizeof(int));
  p->bytes = at;
  return LQ_OK;
}

// The arguments of a call.
struct Call {
  const void *x, *a, *b, *ids, *y;
  void *out, *scratch;
  const int* ranks;
  const float* scales;
  long ldx, ldy, ldo;
  int T, K, L, ids_64;
  const int* widths;
  int n_slices;
  cudaStream_t st;
  int* status;
  int* order(const Plan& p) const { return reinterpret_cast<int*>(static_cast<char*>(scratch) + p.order_at); }
  Tile* tiles(const Plan& p) const { return reinterpret_cast<Tile*>(static_cast<char*>(scratch) + p.tiles_at); }
  int* done(const Plan& p) const { return reinterpret_cast<int*>(static_cast<char*>(scratch) + p.done_at); }
  float* up(const Plan& p) const { return reinterpret_cast<float*>(static_cast<char*>(scratch) + p.up_at); }
  template <typename T> T* vv(const Plan& p) const { return reinterpret_cast<T*>(static_cast<char*>(scratch) + p.vv_at); }
};

// Slices cut into parts of `columns`.
Slices slices_of(const Call& c, int columns) {
  Slices s = {};
  s.n = c.n_slices;
  for (int i = 0; i < c.n_slices; ++i) {
    s.start[i + 1] = s.start[i] + c.widths[i];
    s.part[i + 1] = s.part[i] + (c.widths[i] + columns - 1) / columns;
  }
  s.N = s.start[s.n], s.parts = s.part[s.n];
  return s;
}

// A launch of `bytes` of dynamic shared memory.  Up to 48 KB, static shared memory with it (these kernels have less than 1 KB), needs no leave;
// above, the kernel's limit goes to `most`, what its largest call takes: the limit is the kernel's, so a smaller one, set for
// another host thread's call, could come between a call's own and its launch.
template <typename F>
cudaError_t allow_smem(F* kernel, size_t bytes, size_t most) {
  return bytes > 47 * 1024 ? cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most) : cudaSuccess;
}

template <typename T, int RT>
cudaError_t launch_shrink(const Plan& p, const Call& c) {
  const size_t smem = Shrink<RT>::kBytes;
  cudaError_t e = allow_smem(adapter_shrink_kernel<T, RT>, smem, smem);
  if (e != cudaSuccess) return e;
  return launch_overlapped(adapter_shrink_kernel<T, RT>, dim3(p.max_tiles, (p.R + RT * 16 - 1) / (RT * 16), p.planes),
                           dim3(kShrinkThreads), smem, c.st, static_cast<const T*>(c.x), c.ldx, static_cast<const T*>(c.a), c.ranks,
                           static_cast<const int*>(c.order(p)), static_cast<const Tile*>(c.tiles(p)), c.done(p),
                           static_cast<float*>(c.scratch), c.vv<T>(p), c.up(p), c.T, c.K, p.R, p.rp, p.k_range);
}

template <typename T, typename Y, int KT, int MT>
cudaError_t launch_expand(const Plan& p, const Call& c) {
  using E = Expand<Y, KT, MT>;
  const Slices slices = slices_of(c, 128 * MT);
  const size_t smem = (size_t)E::kStages * E::kStage;
  cudaError_t e = allow_smem(adapter_expand_kernel<T, Y, KT, MT>, smem, smem);
  if (e != cudaSuccess) return e;
  // as many tiles for a CTA as leave a few CTAs for every SM
  const long work = (long)p.max_tiles * slices.parts, slots = (long)sm_count() * 4;
  const int each = work < slots ? 1 : (int)(work / slots);
  return launch_overlapped(adapter_expand_kernel<T, Y, KT, MT>, dim3(slices.parts, (p.max_tiles + each - 1) / each), dim3(256), smem,
                           c.st, static_cast<const Y*>(c.y), c.ldy, static_cast<Y*>(c.out), c.ldo, static_cast<const T*>(c.b),
                           c.ranks, c.scales, static_cast<const int*>(c.order(p)), static_cast<const Tile*>(c.tiles(p)),
                           static_cast<const T*>(c.vv<T>(p)), static_cast<const float*>(c.up(p)), c.T, p.rp, p.max_tiles, each,
                           slices, c.status);
}

template <typename T, typename Y>
cudaError_t run_expand(const Plan& p, const Call& c) {
  if (p.rp <= 16) return launch_expand<T, Y, 1, 4>(p, c);
  if (p.rp <= 32) return launch_expand<T, Y, 2, 4>(p, c);
  if (p.rp <= 64) return launch_expand<T, Y, 4, 4>(p, c);
  if (p.rp <= 128) return launch_expand<T, Y, 8, 4>(p, c);
  return launch_expand<T, Y, 16, 2>(p, c);
}

template <typename T, typename Y, int RT, int KT>
cudaError_t launch_few(const Plan& p, const Call& c) {
  auto bytes = [](size_t R) {
    const size_t halves = 8 * (R / 4 + 1) * 16, sums = (size_t)8 * 16 * RT * 8 * sizeof(float);
    return 2 * R * 8 * sizeof(float) + (halves > sums ? halves : sums);
  };
  const size_t smem = bytes(p.R);
  auto kernel = adapter_few_kernel<T, Y, RT, KT>;
  cudaError_t e = allow_smem(kernel, smem, bytes(kFewRanks));
  if (e != cudaSuccess) return e;
  // as many CTAs for a row as all of them together fit on the SMs, two each
  int ctas = 8;
  while (ctas > 1 && (long)ctas * c.T > 2 * sm_count()) ctas /= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas, c.T);
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = c.st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<const T*>(c.x), c.ldx, static_cast<const Y*>(c.y), c.ldy, static_cast<Y*>(c.out),
                            c.ldo, static_cast<const T*>(c.a), static_cast<const T*>(c.b), c.ranks, c.scales, c.ids, c.ids_64 != 0,
                            c.T, c.K, c.L, p.R, p.rp, slices_of(c, 64));
}

template <typename T>
cudaError_t run_add(const Plan& p, const Call& c, int y_f32) {
  // One launch for few rows.  At 4096 -> 6144 and rank 16 (rows of one adapter / of as many as there are rows), against the three
  // kernels: 1 row 10 us (13), 32 rows 11 / 14 (17 / 26), 64 rows 14 / 16 (25 / 43), 128 rows 20 / 23 (25 / 44).  Every cluster goes over all
  // columns, so with 28672 of them 64 rows take 29 / 33 (22 / 54) and 128 rows 52 / 57 (27 / 57).  What the rule costs: the ids are not
  // known here, nor does it ask for the rank, and every eight rows of one adapter read its matrices again.  64 (65) rows of one adapter /
  // of their own, slices x rank, columns: 1 x 64, 28672: 58 / 71 us (32 / 118); 2 x 256, 28672: 197 / 265 (61 / 482); 128 (129) rows:
  // 1 x 256, 8192: 130 / 170 (78 / 410); 2 x 256, 4096: 116 / 160 (80 / 388).  Rows of their own gain where those of one lose.
  long N = 0;
  for (int i = 0; i < c.n_slices; ++i) N += c.widths[i];
  if ((c.T <= 64 || (c.T <= 128 && N <= 8192)) && p.R <= kFewRanks) {
    if (p.R <= 16) return y_f32 ? launch_few<T, float, 1, 1>(p, c) : launch_few<T, T, 1, 1>(p, c);
    if (p.rp <= 16) return y_f32 ? launch_few<T, float, 4, 1>(p, c) : launch_few<T, T, 4, 1>(p, c);
    return y_f32 ? launch_few<T, float, 4, 4>(p, c) : launch_few<T, T, 4, 4>(p, c);
  }
  const size_t smem = (size_t)(3 * c.L + 5) * sizeof(int);
  cudaError_t e = allow_smem(adapter_plan_kernel, smem, (size_t)(3 * kMaxSlots + 5) * sizeof(int));
  if (e != cudaSuccess) return e;
  e = launch_overlapped(adapter_plan_kernel, dim3(1), dim3(1024), smem, c.st, c.ids, c.ids_64 != 0, c.T, c.L, c.y != c.out, c.order(p), c.tiles(p), c.done(p), p.max_tiles);
  if (e != cudaSuccess) return e;
  if (p.R <= 16) e = launch_shrink<T, 1>(p, c);
  else e = launch_shrink<T, 2>(p, c);
  if (e != cudaSuccess) return e;
  return y_f32 ? run_expand<T, float>(p, c) : run_expand<T, T>(p, c);
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
  long N = 0;
  for (int s = 0; s < n_slices; ++s) {
    if (widths[s] <= 0) return LQ_ERR_BAD_ARG;
    if (widths[s] % 8 || widths[s] > (1 << 22)) return LQ_ERR_SHAPE;
    N += widths[s];
  }
  const int wide = y_f32 ? 4 : 2;
  auto odd = [](const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15) != 0; };
  if (odd(x) || odd(a) || odd(b) || odd(y) || odd(out) || ldx % 8 || ldx < 0 || (ldy * wide) % 16 || (ldo * wide) % 16 ||
      (T > 1 && (ldy < N || ldo < N)) || N > 1 << 22)
    return LQ_ERR_SHAPE;
  if (!scratch || odd(scratch) || scratch_bytes < p.bytes) return LQ_ERR_WORKSPACE;
  const Call c = {x, a, b, ids, y, out, scratch, ranks, scales, ldx, ldy, ldo, T, K, L, ids_64, widths, n_slices, as_stream(stream), status_word()};
  if (!c.status) return LQ_ERR_CUDA;
  const cudaError_t e = dtype == LQ_DT_BF16 ? run_add<__nv_bfloat16>(p, c, y_f32) : run_add<__half>(p, c, y_f32);
  if (e != cudaSuccess) {
    record_cuda_error(e, "adapters_add");
    return LQ_ERR_CUDA;
  }
  return check_launch("adapters_add");
}
