// Grouped W4A8 / INT8 product of a mixture-of-experts layer: for every tile of up to BN sorted activation rows of one
// expert, out = rows x weights(expert)^T in exact int32, then one of three epilogues (see OutMode).
//
// The kernel is the two-CTAs-per-SM tile kernel of the dense linear (lq_gemm_tile.cu) made persistent: the number of tiles is
// known on the device only (it depends on how the tokens chose), so CTA b takes work items b, b + grid, ... of the plan's
// tiles x channel blocks x k-ranges and its rings run on from one item to the next: the copies and the unpacking of the next
// item start while the sums of the last one are read out.  Item order: channel blocks fastest, so that the
// CTAs at work at one time share a few row tiles, and the row tiles of one expert follow each other and find its weights in L2.
// With few rows an expert the k-steps of all tiles may be dealt out in equal shares instead (cut_evenly says when): the two parts of a tile
// that a share's end cuts are joined by whichever CTA comes second, through global memory, and nobody waits.
//
// A tile's width is what its rows need: the MMA's N is its rows in steps of 16 or 32, and the rows come in one box of BN or BN / 2
// rows (one copy a k-step).  Rows of the box behind the tile's are those of the next expert, or zeros; their sums
// are not stored.
//
// Per CTA: warp 0 = copies (8704-byte bulk copy of a blob tile, or a 128 x 128 box of INT8 weights; boxes of rows), warp 1 =
// tensor-memory allocation and MMA issue; with 4-bit weights warps 2..5 and 6..9 = two sets that unpack alternate k-steps into
// tensor memory and warps 10..13 the epilogue, with INT8 weights warps 2..5 and 6..9 two epilogue groups.  The epilogue of an item
// (3 us for 16 rows with the gated activation: one warp's chain of latencies) runs beside the next item's main loop; with
// the sets doing it themselves the weight stream stood still meanwhile (28672 x 4096, eight experts: 4 of 14 us per item).
// Bound by the weights' stream with few rows: one expert of 37888 x 8192 (two items' k-steps a SM at all times) 29 us for 165 MB, 5.7
// TB/s with start and end, 7 TB/s between (362 ns a pair of k-steps); what is left is the start (2 us to the first sums' operands),
// the last round and the join.  One token through two of eight experts' 28672 x 4096: 28 us with the pass before it; the floor is 19.
// A CTA alone on its SM takes 178 ns a k-step (unpacking, and the chain of waits from copy to MMA).
// The stage counts are even wherever two sets take turns, so that a set sees every use of its stages.  All waits are bounded;
// status codes 161-166.
#include <cuda.h>

#include <mutex>

#include "lq_experts.cuh"
#include "lq_experts_epi.cuh"
#include "lq_sched.cuh"
#include "lq_tc_ptx.cuh"

namespace lq {

int make_byte_matrix_map(CUtensorMap* map, const void* ptr, long rows, long row_bytes, int box_rows,
                         int box_bytes);  // lq_gemm_tc.cu

namespace experts {

constexpr int kBlobTile = 8704;
constexpr int kSets = 2;                    // unpacking sets of four warps
constexpr int kNT = 4;                      // operand stages in tensor memory (4-bit weights)
constexpr uint64_t kWaitLimitNs = 2000000000ull;

struct Args {
  const uint8_t* blob;
  const float* s1;
  const float* ascale;
  const int* counts;
  const int4* tiles;
  const int* pair_of_pos;
  EpiArgs epi;
  int4* join;      // of the plan, for this product
  int32_t* part;
  int* status;
  int N, kt_total, n_tiles, which;
};

template <int BN, int NS, bool W4>
struct Cfg {
  static constexpr int kGroups = W4 ? 1 : 2;                  // epilogue groups of four warps
  static constexpr int kThreads = 64 + 128 * ((W4 ? kSets : 0) + kGroups);
  static constexpr int kStep = BN >= 64 ? 32 : 16;            // of the MMA's N
  static constexpr int kXStage = BN * 128;
  static constexpr int kWStage = W4 ? kBlobTile : 128 * 128;
  static constexpr int kAcc = BN <= 64 || !W4 ? 2 : 1;        // accumulators
  static constexpr int kCols = kAcc * BN + (W4 ? 32 * kNT : 0);
  static constexpr int kTmemCols = kCols <= 32 ? 32 : kCols <= 64 ? 64 : kCols <= 128 ? 128 : 256;
  static constexpr int kNumBars = 2 * NS + 2 * kNT + 2 * kAcc;
  static constexpr int kRowInfo = 4 * BN;                     // per warp: scale and destination of the rows it stores
  static constexpr int kSmemBytes = 1024 /* alignment slack */ + NS * (kXStage + kWStage) + kNumBars * 8 + 16 + kRowInfo * 8;
  static_assert(kCols <= 256, "two CTAs per SM share 512 columns");
  static_assert(!W4 || NS % kSets == 0, "a set must see every use of its stages");
  static_assert(2 * (kSmemBytes + 1024) <= 233472, "two CTAs per SM");
};

// One work item: k-steps [kb, ke) of channel block nt for the rows [row0, row0 + rows) of an expert.
struct Item {
  int expert, row0, rows, nt, s, kb, ke;
};
__device__ __forceinline__ Item item_of(const Args& a, int splits, int i, const int4& tile) {
  Item it;
  const int in = i % (a.n_tiles * splits);
  it.s = in / a.n_tiles;
  it.nt = in - it.s * a.n_tiles;
  it.expert = tile.x;
  it.row0 = tile.y;
  it.rows = tile.z;
  it.kb = (it.s * a.kt_total) / splits;
  it.ke = ((it.s + 1) * a.kt_total) / splits;
  return it;
}
__device__ __forceinline__ int4 tile_of(const Args& a, int splits, int i) { return __ldcg(a.tiles + i / (a.n_tiles * splits)); }

// What a CTA has to do: the items blockIdx.x, blockIdx.x + grid, ... of all, or (`even`: k dealt out evenly, EVEN: that may be) the
// k-steps [at, end) of all tiles in a row, whose first and last item may be parts.
template <bool EVEN>
struct Walk {
  int at, end;
  bool even;
  __device__ __forceinline__ Walk(const Args& a, bool dealt, int items) : at(blockIdx.x), end(items), even(EVEN && dealt) {
    if (even) {
      const int total = items * a.kt_total, share = total / (int)gridDim.x, rest = total - share * (int)gridDim.x;
      at = (int)blockIdx.x * share + ((int)blockIdx.x < rest ? (int)blockIdx.x : rest);
      end = at + share + ((int)blockIdx.x < rest ? 1 : 0);
    }
  }
  __device__ __forceinline__ bool more() const { return at < end; }
  __device__ __forceinline__ int number(const Args& a) const { return even ? at / a.kt_total : at; }
  __device__ __forceinline__ Item item(const Args& a, int splits, const int4& tile) const {
    const int i = number(a);
    Item it = item_of(a, splits, i, tile);
    if (even) {
      it.kb = at - i * a.kt_total;
      it.ke = it.kb + (end - at) < a.kt_total ? it.kb + (end - at) : a.kt_total;
    }
    return it;
  }
  __device__ __forceinline__ Item item(const Args& a, int splits) const { return item(a, splits, tile_of(a, splits, number(a))); }
  __device__ __forceinline__ void over(const Item& it) { at += even ? it.ke - it.kb : (int)gridDim.x; }
};

// The other part's sums of (up to) sixteen rows.
__device__ __forceinline__ void add_part(int (&v)[16], const int32_t* other, int rows) {
#pragma unroll
  for (int j = 0; j < 16; ++j)
    if (j < rows) v[j] += __ldcg(other + j * 128);
}

template <int BN, int NS, bool W4, int MODE, bool EVEN>
__global__ void __launch_bounds__(Cfg<BN, NS, W4>::kThreads, 2)
experts_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_xhalf,
               const __grid_constant__ CUtensorMap tmap_w, const Args args) {
  using C = Cfg<BN, NS, W4>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t base = (raw_addr + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - raw_addr);

  const uint32_t xs = base;                                   // NS row stages (1024-aligned, 128-byte swizzle)
  const uint32_t ws = xs + NS * C::kXStage;                   // NS weight stages (1024-aligned for INT8: swizzled too)
  const uint32_t bars = ws + NS * C::kWStage;
  const uint32_t bar_full = bars;                             // [NS] copies landed
  const uint32_t bar_empty = bar_full + NS * 8;               // [NS] stage may be overwritten
  const uint32_t bar_aready = bar_empty + NS * 8;             // [kNT] operand in tensor memory
  const uint32_t bar_afree = bar_aready + kNT * 8;            // [kNT] MMAs that read the operand are done
  const uint32_t bar_accfull = bar_afree + kNT * 8;           // [kAcc] sums final
  const uint32_t bar_accfree = bar_accfull + C::kAcc * 8;     // [kAcc] sums read out
  const uint32_t tmem_slot = bar_accfree + C::kAcc * 8;
  volatile uint32_t* tmem_slot_p = reinterpret_cast<volatile uint32_t*>(smem + (tmem_slot - base));
  float* row_scale = reinterpret_cast<float*>(smem + (tmem_slot + 16 - base));   // [epilogue warp][BN / kGroups]
  int* row_pair = reinterpret_cast<int*>(row_scale + C::kRowInfo);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < NS; ++s) {
      ptx::mbar_init(bar_full + 8 * s, 1);
      ptx::mbar_init(bar_empty + 8 * s, W4 ? 129 : 1);
    }
    for (int t = 0; t < kNT; ++t) {
      ptx::mbar_init(bar_aready + 8 * t, 128);
      ptx::mbar_init(bar_afree + 8 * t, 1);
    }
    for (int b = 0; b < C::kAcc; ++b) {
      ptx::mbar_init(bar_accfull + 8 * b, 1);
      ptx::mbar_init(bar_accfree + 8 * b, 4 * C::kGroups);   // one arrival per epilogue warp
    }
    ptx::fence_mbar_init();
    ptx::prefetch_tensormap(&tmap_x);
    ptx::prefetch_tensormap(&tmap_xhalf);
    if (!W4) ptx::prefetch_tensormap(&tmap_w);
  }
  if (warp == 1) {
    ptx::tmem_alloc(tmem_slot, C::kTmemCols);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  allow_dependents();
  dependency_wait();   // the plan, the rows and the buffers written here belong to earlier kernels until now
  const uint32_t tmem_acc = *tmem_slot_p;
  const uint32_t tmem_a = tmem_acc + C::kAcc * BN;
  // Where k is whole the first tile's entry is requested together with the number of tiles: the table has room for every tile that
  // a launch of this grid can have, so an entry that is not there is read as anything and not used.
  int4 tile = make_int4(0, 0, 0, 0);
  if (MODE != kOutPlanes && warp == 0) tile = tile_of(args, 1, blockIdx.x);
  const int4 counts = __ldcg(reinterpret_cast<const int4*>(args.counts));
  const int cuts = args.which == 0 ? counts.z : counts.w;
  const int splits = MODE != kOutPlanes ? 1 : cuts;
  const int items = counts.x * args.n_tiles * splits;
  const bool dealt = EVEN && cuts == 0;

  if (warp == 0) {
    // ------------------------------------------------------------------ copies
    // The whole warp walks the loop and one elected lane issues, as with the MMAs (see ptx::elect_one): a loop that only thread 0
    // walks takes about 450 cycles a k-step.
    const bool leader = ptx::elect_one();
    Ring<NS> ring;
    int issued = 0;
    bool ok = true;
    for (Walk<EVEN> w(args, dealt, items); ok && w.more();) {
      if (MODE == kOutPlanes || w.even || w.at != (int)blockIdx.x) tile = tile_of(args, splits, w.number(args));
      const Item it = w.item(args, splits, tile);
      w.over(it);
      const bool few = it.rows <= BN / 2;
      const uint32_t tx = (uint32_t)((few ? BN / 2 : BN) * 128 + C::kWStage);
      const uint8_t* src = W4 ? args.blob + ((size_t)((size_t)it.expert * args.n_tiles + it.nt) * args.kt_total + it.kb) * kBlobTile : nullptr;
      const int wrow = W4 ? 0 : it.expert * args.N + it.nt * 128;
      for (int kt = it.kb; kt < it.ke; ++kt) {
        ok = ptx::mbar_wait_bounded(bar_empty + 8 * ring.s, ring.ph ^ 1u, kWaitLimitNs);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) {
          if (leader) atomicExch(args.status, 161);
          break;
        }
        const uint32_t full = bar_full + 8 * ring.s;
        const uint32_t wdst = ws + ring.s * C::kWStage, xdst = xs + ring.s * C::kXStage;
        if (leader) {
          ptx::mbar_expect_tx(full, tx);
          if (W4) ptx::bulk_load(wdst, src, kBlobTile, full);
          else ptx::tensor_load_2d(wdst, &tmap_w, kt * 128, wrow, full);
          ptx::tensor_load_2d(xdst, few ? &tmap_xhalf : &tmap_x, kt * 128, it.row0, full);
        }
        if (W4) src += kBlobTile;
        ring.advance();
        ++issued;
      }
    }
    if (!ok) {
      // copies already issued still write shared memory: let them land before the CTA exits
      for (int q = issued > NS ? issued - NS : 0; q < issued; ++q)
        ptx::mbar_wait_bounded(bar_full + 8 * (q % NS), (uint32_t)(q / NS) & 1u, kWaitLimitNs);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issue
    // The whole warp walks the loop; one elected lane issues (see ptx::elect_one).
    const bool leader = ptx::elect_one();
    Ring<NS> ring;
    Ring<kNT> tring;
    Ring<C::kAcc> accring;
    bool ok = true;
    for (Walk<EVEN> w(args, dealt, items); ok && w.more();) {
      const Item it = w.item(args, splits);
      w.over(it);
      const uint32_t idesc = ptx::idesc_i8((it.rows + C::kStep - 1) / C::kStep * C::kStep);
      ok = ptx::mbar_wait_bounded(bar_accfree + 8 * accring.s, accring.ph ^ 1u, kWaitLimitNs);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) {
        if (leader) atomicExch(args.status, 162);
        break;
      }
      ptx::tc_fence_after();
      const uint32_t acc = tmem_acc + accring.s * BN;
      for (int kt = it.kb; kt < it.ke; ++kt) {
        // 4-bit weights: "operand ready" implies that the rows have landed (every unpacking thread saw its stage's full barrier, weights and
        // rows, before it made the operand)
        ok = W4 ? ptx::mbar_wait_bounded(bar_aready + 8 * tring.s, tring.ph, kWaitLimitNs)
                : ptx::mbar_wait_bounded(bar_full + 8 * ring.s, ring.ph, kWaitLimitNs);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) {
          if (leader) atomicExch(args.status, 163);
          break;
        }
        ptx::tc_fence_after();
        const uint32_t xb = xs + ring.s * C::kXStage;
        const uint32_t wb = ws + ring.s * C::kWStage;
        const uint32_t ab = tmem_a + tring.s * 32;
        if (leader) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint64_t bdesc = ptx::smem_desc_sw128(xb + j * 32);
            const uint32_t accumulate = (kt > it.kb || j > 0) ? 1u : 0u;
            if (W4) ptx::mma_i8_ts(acc, ab + j * 8, bdesc, idesc, accumulate);
            else ptx::mma_i8_ss(acc, ptx::smem_desc_sw128(wb + j * 32), bdesc, idesc, accumulate);
          }
          ptx::tc_commit(bar_empty + 8 * ring.s);
          if (W4) ptx::tc_commit(bar_afree + 8 * tring.s);
        }
        ring.advance();
        tring.advance();
      }
      if (ok && leader) ptx::tc_commit(bar_accfull + 8 * accring.s);
      accring.advance();
    }
  } else if (W4 && warp < 2 + 4 * kSets) {
    // ------------------------------------------------------------------ unpacking
    const int quad = warp & 3;               // TMEM lane quadrant this warp may access
    const int row = quad * 32 + lane;        // channel inside the block == TMEM lane
    const uint32_t lane_addr = (uint32_t)(quad * 32) << 16;
    const int set = (warp - 2) >> 2;
    Ring<NS> ring;
    Ring<kNT> tring;
    int turn = 0;
    bool ok = true;
    for (Walk<EVEN> w(args, dealt, items); ok && w.more();) {
      const Item it = w.item(args, splits);
      w.over(it);
      // The set walks its own steps alone: with the other set's as iterations that do nothing the unpacking warps' issue slots cost
      // 4 % at one token.
      const int steps = it.ke - it.kb;
      const int skip = turn ^ set;         // the item's first step is the other set's
      turn ^= steps & 1;
      if (skip) {
        ring.advance();
        tring.advance();
      }
      for (int q = skip; q < steps; q += kSets) {
        if (!ptx::mbar_wait_bounded(bar_full + 8 * ring.s, ring.ph, kWaitLimitNs)) {
          atomicExch(args.status, 164);
          ok = false;
          break;
        }
        const uint8_t* wst = smem + (ws - base) + ring.s * C::kWStage;
        uint4 ch[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) ch[c] = *reinterpret_cast<const uint4*>(wst + (c * 128 + row) * 16);
        const uint32_t meta = *reinterpret_cast<const uint32_t*>(wst + 8192 + row * 4);
        ptx::mbar_arrive(bar_empty + 8 * ring.s);
        uint32_t v[32];
        unpack_row(ch, meta, v);
        if (!ptx::mbar_wait_bounded(bar_afree + 8 * tring.s, tring.ph ^ 1u, kWaitLimitNs)) {
          atomicExch(args.status, 165);
          ok = false;
          break;
        }
        __syncwarp();   // lanes leave the poll loops one by one; tcgen05.st / wait::st need the warp converged
        ptx::tc_fence_after();
        ptx::tmem_st32(tmem_a + lane_addr + tring.s * 32, v);
        ptx::tc_wait_st();
        ptx::tc_fence_before();
        ptx::mbar_arrive(bar_aready + 8 * tring.s);
        // own stages are every second one (both rings have an even number): step over the other set's
        const bool two = q + 1 < steps;
        ring.s += two ? 2 : 1;
        if (ring.s >= NS) ring.s -= NS, ring.ph ^= 1u;
        tring.s += two ? 2 : 1;
        if (tring.s >= kNT) tring.s -= kNT, tring.ph ^= 1u;
      }
    }
  } else {
    // ------------------------------------------------------------------ epilogue
    constexpr int kFirst = 2 + (W4 ? 4 * kSets : 0), kRows = BN / C::kGroups;
    const int quad = warp & 3;               // TMEM lane quadrant this warp may access
    const int row = quad * 32 + lane;        // channel inside the block == TMEM lane
    const uint32_t lane_addr = (uint32_t)(quad * 32) << 16;
    const int group = (warp - kFirst) >> 2;
    float* sc = row_scale + (warp - kFirst) * kRows;   // rows 16 (kGroups i + group) + (0..15) at 16 i
    int* pair = row_pair + (warp - kFirst) * kRows;
    Ring<C::kAcc> accring;
    bool ok = true;
    for (Walk<EVEN> w(args, dealt, items); ok && w.more();) {
      const Item it = w.item(args, splits);
      w.over(it);
      // What the epilogue needs beside the sums is requested ahead of them: behind the last MMA it would wait for the weight copies
      // of the next item, which fill the queues to memory (a channel scale read there cost 3 to 5 us an item).
      const int n = it.nt * 128 + row;
      const bool n_ok = n < args.N;
      float w_scale = 0.f;
      if (MODE != kOutPlanes) {
        if (n_ok) w_scale = args.s1[(size_t)it.expert * args.N + n];
        __syncwarp();   // every lane is done with the last item's rows
#pragma unroll
        for (int q = lane; q < kRows; q += 32) {
          const int r = 16 * (C::kGroups * (q >> 4) + group) + (q & 15);
          const bool in = r < it.rows;
          sc[q] = in ? args.ascale[it.row0 + r] : 0.f;
          if (MODE == kOutPairs) pair[q] = in ? args.pair_of_pos[it.row0 + r] : 0;
        }
        __syncwarp();
      }
      // A part of a tile: this warp's sums go to memory, and the warp that comes second (the other CTA's, for the same channels and
      // rows) adds both; it finds out ahead of its own sums, if it can.  Nobody waits.
      const bool part = EVEN && it.ke - it.kb < args.kt_total;
      const int side = it.kb > 0 ? 1 : 0, cut = (int)blockIdx.x - side;   // between the CTAs `cut` and `cut` + 1
      int* here = reinterpret_cast<int*>(args.join + cut) + (warp - kFirst);
      bool second = false;
      if (part) {
        int before = 0;
        if (lane == 0) before = *reinterpret_cast<volatile int*>(here);
        second = __shfl_sync(0xffffffffu, before, 0) != 0;
        __threadfence();
      }
      if (!ptx::mbar_wait_bounded(bar_accfull + 8 * accring.s, accring.ph, kWaitLimitNs)) {
        atomicExch(args.status, 166);
        ok = false;
      }
      // the warp reads tensor memory and shuffles as one: it goes on as one or not at all
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      ptx::tc_fence_after();
      const uint32_t acc = tmem_acc + accring.s * BN + lane_addr;
      if (part && !second) {
        int32_t* mine = args.part + (size_t)((2 * cut + side) * BN) * 128 + row;
#pragma unroll 1
        for (int c0 = 0; c0 < it.rows; c0 += 16) {
          int v[16];
          ptx::tmem_ld16(acc + c0, v);
          ptx::tc_wait_ld();
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (c0 + j < it.rows) mine[(c0 + j) * 128] = v[j];
        }
        __threadfence();
        __syncwarp();
        int before = 0;
        if (lane == 0) before = atomicAdd(here, 1);
        second = __shfl_sync(0xffffffffu, before, 0) != 0;
        __threadfence();
      }
      const int rows = part && !second ? 0 : it.rows;
#pragma unroll 1
      for (int c0 = 16 * group, at = 0; c0 < rows; c0 += 16 * C::kGroups, at += 16) {
        int v[16];
        ptx::tmem_ld16(acc + c0, v);
        ptx::tc_wait_ld();
        if (part) add_part(v, args.part + (size_t)((2 * cut + 1 - side) * BN + c0) * 128 + row, it.rows - c0);
        store_rows<MODE>(args.epi, v, (long)it.row0 + c0, it.rows - c0, n, n_ok, w_scale, sc + at, pair + at, it.s);
      }
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(bar_accfree + 8 * accring.s);
      accring.advance();
    }
  }

  __syncwarp();
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem_acc, C::kTmemCols);
  }
}

template <int BN, int NS, bool W4, int MODE, bool EVEN = false>
static int launch_mode(const Product& p, const Plan& plan, cudaStream_t st) {
  using C = Cfg<BN, NS, W4>;
  auto kern = &experts_kernel<BN, NS, W4, MODE, EVEN>;
  static std::once_flag once[64];
  int dev = 0;
  cudaGetDevice(&dev);
  cudaError_t attr_err = cudaSuccess;
  std::call_once(once[dev & 63], [&]() {
    attr_err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes);
  });
  if (attr_err != cudaSuccess) {
    record_cuda_error(attr_err, "cudaFuncSetAttribute(experts_kernel)");
    return LQ_ERR_CUDA;
  }
  CUtensorMap tx, txh, tw;
  if (int rc = make_byte_matrix_map(&tx, p.x, p.rows, p.K, BN, 128)) return rc;
  if (int rc = make_byte_matrix_map(&txh, p.x, p.rows, p.K, BN / 2, 128)) return rc;
  if (W4) tw = tx;
  else if (int rc = make_byte_matrix_map(&tw, p.w, (long)p.E * p.N, p.K, 128, 128)) return rc;
  Args a;
  a.blob = static_cast<const uint8_t*>(p.w);
  a.s1 = p.s1;
  a.ascale = p.ascale;
  a.counts = plan.counts;
  a.tiles = plan.tiles;
  a.pair_of_pos = plan.pair_of_pos;
  a.epi.out = p.out;
  a.epi.amax = p.amax;
  a.epi.rows = p.rows;
  a.epi.N = p.N;
  a.epi.out_dtype = p.out_dtype;
  a.join = plan.join[p.which];
  a.part = plan.part;
  a.status = status_word();
  a.N = p.N;
  a.kt_total = p.K / 128;
  a.n_tiles = (p.N + 127) / 128;
  a.which = p.which;
  if (!a.status) return LQ_ERR_CUDA;
  const long items = max_tiles(p.rows, p.E, plan.bn) * a.n_tiles * (MODE == kOutPlanes ? plan.rule[p.which].most : 1);
  const long slots = plan.slots;
  const cudaError_t e = launch_overlapped(kern, dim3((unsigned)(items < slots ? items : slots)), dim3(C::kThreads),
                                          (size_t)C::kSmemBytes, st, tx, txh, tw, a);
  if (e != cudaSuccess) {
    record_cuda_error(e, "experts_kernel launch");
    return LQ_ERR_CUDA;
  }
  return check_launch("experts_kernel");
}

template <int BN, int NS, bool W4>
static int launch_product(const Product& p, const Plan& plan, cudaStream_t st) {
  if (p.out_mode == kOutPlanes) return launch_mode<BN, NS, W4, kOutPlanes>(p, plan, st);
  if constexpr (W4 && BN == kEvenRows) {
    if (plan.rule[p.which].even)
      return p.out_mode == kOutPairs ? launch_mode<BN, NS, W4, kOutPairs, true>(p, plan, st)
                                     : launch_mode<BN, NS, W4, kOutGated, true>(p, plan, st);
  }
  if (p.out_mode == kOutPairs) return launch_mode<BN, NS, W4, kOutPairs>(p, plan, st);
  return launch_mode<BN, NS, W4, kOutGated>(p, plan, st);
}

int run_product(const Product& p, const Plan& plan, cudaStream_t st) {
  if (plan.bn > 128) return run_product_pair(p, plan, st);
  if (p.w_kind == kBlob) {
    switch (plan.bn) {
      case 32: return launch_product<32, 8, true>(p, plan, st);
      case 64: return launch_product<64, 6, true>(p, plan, st);
      default: return launch_product<128, 4, true>(p, plan, st);
    }
  }
  switch (plan.bn) {
    case 32: return launch_product<32, 5, false>(p, plan, st);
    case 64: return launch_product<64, 4, false>(p, plan, st);
    default: return launch_product<128, 3, false>(p, plan, st);
  }
}

}  // namespace experts
}  // namespace lq
