// Grouped W4A8 / INT8 product for experts with many rows: CTA pairs, tcgen05.mma.cta_group::2 on tiles of 256 channels x up to 192
// (4-bit weights) or 256 (INT8) sorted rows of one expert.  The reasons for pairs are those of the dense pair kernels
// (lq_gemm_pair.cu, lq_i8_pair.cu): a one-CTA tile kernel at its full MMA rate would need more bytes per clock than L2
// delivers, and two CTAs that share the rows' tile need 0.6 of them.
//
// Work: pair p of P takes the tiles p, p + P, ... of the plan's row tiles x 256-channel blocks, in groups of eight row tiles (see
// tile_coords), so that the tiles at work at one time share rows and weights in L2.  How many there are is known on the device
// only.  A tile's MMA is as wide as its rows need, in steps of 32; each CTA stages half of them in ONE box, for which there is a tensor
// map of every width (boxes of 64 and 16 rows as needed: 28 % slower on full tiles of 192, the copies are bound by their number).
// Rows of the box behind the tile's are those of the next expert, or zeros; their sums are not stored.  With an odd number of 128-channel blocks the
// second CTA's half of the last tile lies behind the expert's channels: it computes with other weights and stores nothing.
//
// Per CTA, connected by mbarrier rings; rank = CTA's rank in its pair:
//   warp 0   weight producer: 8704-byte bulk copy of a blob tile, or a 128 x 128 box of INT8 weights, per k-step
//   warp 2   row producer
//   warp 3   INT8: relay, tells the leader CTA when both copies of a stage have landed here
//   warp 1   tensor-memory allocation; on rank 0 MMA issue (one elected lane) and commits to the barriers of both CTAs
//   4-bit weights: three unpacking sets of four warps taking the k-steps in turn (the ring of nine stages is a multiple of
//            three, so a set sees every use of its stages; an operand stage is waited for by the set that fills it, and the
//            MMAs of the set's own last step but one are then known to be done), then two epilogue groups
//   INT8:    four epilogue groups
// With 4-bit weights bound by the tensor pipe under the part's power limit and by the unpacking warps' issue slots: 8192 tokens x 2 experts through
// 4096 -> 14336 -> 4096, 5.8 TOP, 2.60 to 2.75 ms with all passes, 2.1 POPS (dense INT8 products hold about 3.05 here); at 2048 tokens the pipe is
// 66 and 71 % busy, the issue slots 62 and 50 %.  INT8 weights, 4000 rows of 14336 to 4096, 0.47 TOP, 250 to 270 us with the rows' quantisation,
// 1.8 POPS: the pipe is 66 % busy, and the dense kernel (lq_i8_pair.cu) takes 158 us for the same product in one matrix, where this one with rows
// that come in INT8 takes 218 to 225 with one expert, 230 to 255 with eight of 500 rows and 270 with uneven ones.  About 25 us of that are the plan
// and the rows' copies, the ends of experts inside tiles are the step from one to eight; the rest is not explained.  Short k is bound by its
// outputs: 13332 rows of 1792 to 4096 in float32 write 218 MB, tensor pipe 43 %.
// Tensor memory (512 columns): two accumulators, and four 32-column operand stages with 4-bit weights.  No load uses cluster
// multicast.  Every wait is bounded; status codes 171-177.
#include <cuda.h>

#include <mutex>

#include "lq_experts.cuh"
#include "lq_experts_epi.cuh"
#include "lq_pair_common.cuh"
#include "lq_sched.cuh"
#include "lq_tc_ptx.cuh"

namespace lq {

int make_byte_matrix_map(CUtensorMap* map, const void* ptr, long rows, long row_bytes, int box_rows,
                         int box_bytes);  // lq_gemm_tc.cu

namespace experts {
namespace pair {

constexpr int kBlobTile = 8704;
constexpr int kNT = 4;
constexpr uint64_t kWaitLimitNs = 2000000000ull;

struct Args {
  const uint8_t* blob;
  const float* s1;
  const float* ascale;
  const int* counts;
  const int4* tiles;
  const int* pair_of_pos;
  EpiArgs epi;
  int* status;
  int N, kt_total, n_tiles, n2_tiles, pairs;   // n_tiles: 128-channel blocks of an expert, n2_tiles: tiles of 256
};

template <bool W4>
struct Cfg {
  static constexpr int kBN = W4 ? kPairRowsBlob : kPairRowsInt8;
  static constexpr int kNS = W4 ? 9 : 6;
  static constexpr int kSets = W4 ? 3 : 0;
  static constexpr int kGroups = W4 ? 2 : 4;
  static constexpr int kThreads = 128 * (1 + kSets + kGroups);
  static constexpr int kXStage = kBN / 2 * 128;
  static constexpr int kWStage = W4 ? kBlobTile : 128 * 128;
  static constexpr int kNumBars = 3 * kNS + 2 * kNT + 4;
  static constexpr int kBarBytes = kNumBars * 8 + 16 + 8 * kGroups;
  static constexpr int kRowInfo = kGroups * 2 * kBN;          // per group, two tiles: scale and destination of every row
  static constexpr int kSmemBytes = 1024 /* alignment slack */ + kNS * (kXStage + kWStage) + ((kBarBytes + 15) & ~15) + kRowInfo * 8;
  static_assert(kSmemBytes <= 232448, "shared memory budget exceeded");
  static_assert(!W4 || kNS % 3 == 0, "a set must see every use of its stages");
  static_assert(2 * kBN + (W4 ? 32 * kNT : 0) <= 512, "tensor memory budget exceeded");
};

// Tensor maps of the rows, x[i] with boxes of 16 (i + 1) rows, and of INT8 weights.
struct Maps {
  CUtensorMap x[kPairRowsInt8 / 32];
  CUtensorMap w;
};

struct Tile {
  int expert, row0, rows, n2;
};
__device__ __forceinline__ Tile tile_at(const Args& a, int i, int row_tiles) {
  Tile t;
  int mt;
  pairc::tile_coords(i, a.n2_tiles, row_tiles, pairc::kGroupM, t.n2, mt);
  const int4 q = __ldcg(a.tiles + mt);
  t.expert = q.x;
  t.row0 = q.y;
  t.rows = q.z;
  return t;
}
__device__ __forceinline__ int width(int rows) { return (rows + 31) & ~31; }

// MODE: kOutPairs or kOutGated (k is whole).
template <bool W4, int MODE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Cfg<W4>::kThreads, 1)
experts_pair_kernel(const __grid_constant__ Maps maps, const Args args) {
  using C = Cfg<W4>;
  constexpr int kNS = C::kNS, kBN = C::kBN;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t base = (raw_addr + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - raw_addr);

  const uint32_t xs = base;                                  // kNS row stages (1024-aligned, 128-byte swizzle)
  const uint32_t ws = xs + kNS * C::kXStage;                 // kNS weight stages
  const uint32_t bars = ws + kNS * C::kWStage;
  const uint32_t bar_full = bars;                            // [kNS] both copies of the stage landed (this CTA)
  const uint32_t bar_empty = bar_full + kNS * 8;             // [kNS] the MMAs that read the stage are done (and its weights unpacked)
  const uint32_t bar_ready = bar_empty + kNS * 8;            // [kNS] INT8, used on rank 0: the stage landed in both CTAs
  const uint32_t bar_aready = bar_ready + kNS * 8;           // [kNT] used on rank 0: operand in the tensor memory of both CTAs
  const uint32_t bar_afree = bar_aready + kNT * 8;           // [kNT] MMAs that read the operand stage are done
  const uint32_t bar_accfull = bar_afree + kNT * 8;          // [2] sums final
  const uint32_t bar_accfree = bar_accfull + 2 * 8;          // [2] used on rank 0: sums read out in both CTAs
  const uint32_t tmem_slot = bar_accfree + 2 * 8;
  uint8_t* gen_bars = smem + (bars - base);
  volatile uint32_t* tmem_slot_p = reinterpret_cast<volatile uint32_t*>(gen_bars + C::kNumBars * 8);
  volatile int* wait_flag = reinterpret_cast<volatile int*>(gen_bars + C::kNumBars * 8 + 16);   // [group][2]
  float* row_scale = reinterpret_cast<float*>(gen_bars + ((C::kBarBytes + 15) & ~15));         // [group][2][kBN]
  int* row_pair = reinterpret_cast<int*>(row_scale + C::kRowInfo);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = ptx::cluster_ctarank();
  const int pair = (int)ptx::cluster_id_x();

  if (threadIdx.x == 0) {
    for (int s = 0; s < kNS; ++s) {
      ptx::mbar_init(bar_full + 8 * s, 2);                   // one expect_tx arrival per producer
      ptx::mbar_init(bar_empty + 8 * s, W4 ? 129 : 1);       // 128 unpacking threads + the MMA thread's commit
      ptx::mbar_init(bar_ready + 8 * s, 2);                  // one relay arrival per CTA
    }
    for (int t = 0; t < kNT; ++t) {
      ptx::mbar_init(bar_aready + 8 * t, 8);                 // one arrival per warp of the owning set, both CTAs
      ptx::mbar_init(bar_afree + 8 * t, 1);
    }
    for (int b = 0; b < 2; ++b) {
      ptx::mbar_init(bar_accfull + 8 * b, 1);
      ptx::mbar_init(bar_accfree + 8 * b, 2 * 4 * C::kGroups);   // one arrival per epilogue warp, both CTAs
    }
    ptx::fence_mbar_init();
    ptx::prefetch_tensormap(&maps.x[kBN / 32 - 1]);
    if (!W4) ptx::prefetch_tensormap(&maps.w);
  }
  if (warp == 1) {
    ptx::tmem_alloc_pair(tmem_slot, 512);
    ptx::tmem_relinquish_pair();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::cluster_sync_all();   // the barriers of both CTAs exist before anything arrives on them from the peer
  ptx::tc_fence_after();
  const uint32_t tmem_base = *tmem_slot_p;
  const uint32_t tmem_a = tmem_base + 2 * kBN;
  const uint32_t leader_ready = ptx::map_to_cta(bar_ready, 0);
  const uint32_t leader_aready = ptx::map_to_cta(bar_aready, 0);
  const uint32_t leader_accfree = ptx::map_to_cta(bar_accfree, 0);
  allow_dependents();
  dependency_wait();   // the plan, the rows and the buffers written here belong to earlier kernels until now
  const int row_tiles = __ldcg(args.counts);
  const int items = row_tiles * args.n2_tiles;

  if (warp == 0 || warp == 2) {
    // ------------------------------------------------------------------ producers
    // As with the MMAs the whole warp walks the loop and one elected lane issues: a loop that only thread 0 walks needed about
    // 450 cycles to issue a k-step's copies, and the rings of the 4-bit kernel, whose k-step is 415 cycles of MMAs, ran dry.
    const bool leader = ptx::elect_one();
    const bool weights = (warp == 0);
    Ring<kNS> ring;
    int issued = 0;
    bool ok = true;
    for (int i = pair; ok && i < items; i += args.pairs) {
      const Tile t = tile_at(args, i, row_tiles);
      const int nt = 2 * t.n2 + (int)rank;
      const uint8_t* wsrc = W4 ? args.blob + ((size_t)t.expert * args.n_tiles + (nt < args.n_tiles ? nt : args.n_tiles - 1)) *
                                                 (size_t)args.kt_total * kBlobTile : nullptr;
      const int half = width(t.rows) / 2;
      const CUtensorMap* xmap = &maps.x[half / 16 - 1];
      const int row0 = weights ? t.expert * args.N + nt * 128 : t.row0 + (int)rank * half;
      for (int kt = 0; kt < args.kt_total; ++kt) {
        ok = ptx::mbar_wait_bounded(bar_empty + 8 * ring.s, ring.ph ^ 1u, kWaitLimitNs);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) {
          if (leader) atomicExch(args.status, 171);
          break;
        }
        const uint32_t full = bar_full + 8 * ring.s;
        if (weights) {
          const uint32_t dst = ws + ring.s * C::kWStage;
          if (leader) {
            ptx::mbar_expect_tx(full, C::kWStage);
            if (W4) ptx::bulk_load(dst, wsrc, kBlobTile, full);
            else ptx::tensor_load_2d(dst, &maps.w, kt * 128, row0, full);
          }
          if (W4) wsrc += kBlobTile;
        } else {
          const uint32_t dst = xs + ring.s * C::kXStage;
          if (leader) {
            ptx::mbar_expect_tx(full, (uint32_t)half * 128u);
            ptx::tensor_load_2d(dst, xmap, kt * 128, row0, full);
          }
        }
        ring.advance();
        ++issued;
      }
    }
    if (!ok) {
      // copies already issued still write shared memory: let them land before the CTA exits
      Ring<kNS> back;
      const int first = issued > kNS ? issued - kNS : 0;
      for (int q = 0; q < issued; ++q) {
        if (q >= first) ptx::mbar_wait_bounded(bar_full + 8 * back.s, back.ph, kWaitLimitNs);
        back.advance();
      }
    }
  } else if (warp == 3) {
    // ------------------------------------------------------------------ relay (one thread; INT8)
    if (!W4 && lane == 0) {
      Ring<kNS> ring;
      bool ok = true;
      for (int i = pair; ok && i < items; i += args.pairs) {
        for (int kt = 0; kt < args.kt_total; ++kt) {
          if (!ptx::mbar_wait_bounded(bar_full + 8 * ring.s, ring.ph, kWaitLimitNs)) {
            atomicExch(args.status, 172);
            ok = false;
            break;
          }
          if (rank == 0) ptx::mbar_arrive(bar_ready + 8 * ring.s);
          else ptx::mbar_arrive_remote(leader_ready + 8 * ring.s);
          ring.advance();
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issue (leader CTA)
    // The whole warp walks the loop; one elected lane issues (see ptx::elect_one).
    if (rank == 0) {
      const bool leader = ptx::elect_one();
      Ring<kNS> ring;
      Ring<kNT> tring;
      Ring<2> accring;
      bool ok = true;
      for (int i = pair; ok && i < items; i += args.pairs) {
        const Tile t = tile_at(args, i, row_tiles);
        const uint32_t idesc = ptx::idesc_i8_pair(width(t.rows));
        if (!ptx::mbar_wait_bounded(bar_accfree + 8 * accring.s, accring.ph ^ 1u, kWaitLimitNs)) {
          if (leader) atomicExch(args.status, 173);
          ok = false;
        }
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        ptx::tc_fence_after();
        const uint32_t tmem_acc = tmem_base + accring.s * kBN;
        for (int kt = 0; kt < args.kt_total; ++kt) {
          // 4-bit weights: "operand ready" from both CTAs implies that the rows of both have landed (every unpacking thread saw
          // its stage's full barrier, weights and rows, before it made the operand)
          const uint32_t bar = W4 ? bar_aready + 8 * tring.s : bar_ready + 8 * ring.s;
          if (!ptx::mbar_wait_bounded(bar, W4 ? tring.ph : ring.ph, kWaitLimitNs)) {
            if (leader) atomicExch(args.status, 174);
            ok = false;
          }
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          ptx::tc_fence_after();
          const uint32_t xb = xs + ring.s * C::kXStage;
          const uint32_t wb = ws + ring.s * C::kWStage;
          const uint32_t ab = tmem_a + tring.s * 32;
          if (leader) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint64_t bdesc = ptx::smem_desc_sw128(xb + j * 32);
              const uint32_t accumulate = (kt > 0 || j > 0) ? 1u : 0u;
              if (W4) ptx::mma_i8_ts_pair(tmem_acc, ab + j * 8, bdesc, idesc, accumulate);
              else ptx::mma_i8_ss_pair(tmem_acc, ptx::smem_desc_sw128(wb + j * 32), bdesc, idesc, accumulate);
            }
            ptx::tc_commit_pair(bar_empty + 8 * ring.s);
            if (W4) ptx::tc_commit_pair(bar_afree + 8 * tring.s);
          }
          ring.advance();
          tring.advance();
        }
        if (ok && leader) ptx::tc_commit_pair(bar_accfull + 8 * accring.s);
        accring.advance();
      }
    }
  } else if (W4 && warp >= 8 && warp < 8 + 4 * C::kSets) {
    // ------------------------------------------------------------------ unpacking (kSets sets, k-steps in turn)
    const int my_set = (warp - 8) >> 2;
    const int quad = warp & 3;               // TMEM lane quadrant this warp may access
    const int row = quad * 32 + lane;        // channel inside the CTA's block == TMEM lane
    const uint32_t lane_addr = (uint32_t)(quad * 32) << 16;
    // A stage of the ring is always the same set's.  An operand stage is not (four, three sets): a set that comes back to one knows by the
    // stages that it waited for before, which the MMAs free in order, that the barrier is at most one phase away.
    // The set walks its own k-steps alone, every kSets-th of all of the pair's. Walking the others' too, as iterations that do
    // nothing, was 3 % slower (8192 tokens: 2.78 ms against 2.70): these warps' issue slots bound the kernel.
    const int tiles = items > pair ? (items - pair + args.pairs - 1) / args.pairs : 0;
    const int steps = tiles * args.kt_total;
    Ring<kNS> ring;
    Ring<kNT> tring;
    ring.s = tring.s = my_set;
    for (int q = my_set; q < steps; q += C::kSets) {
      if (!ptx::mbar_wait_bounded(bar_full + 8 * ring.s, ring.ph, kWaitLimitNs)) {
        atomicExch(args.status, 175);
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
        atomicExch(args.status, 176);
        break;
      }
      __syncwarp();   // lanes leave the poll loops one by one; tcgen05.st / wait::st need the warp converged
      ptx::tc_fence_after();
      ptx::tmem_st32(tmem_a + lane_addr + tring.s * 32, v);
      ptx::tc_wait_st();
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (rank == 0) ptx::mbar_arrive(bar_aready + 8 * tring.s);
        else ptx::mbar_arrive_remote(leader_aready + 8 * tring.s);
      }
      ring.s += C::kSets;
      if (ring.s >= kNS) ring.s -= kNS, ring.ph ^= 1u;
      tring.s += C::kSets;
      if (tring.s >= kNT) tring.s -= kNT, tring.ph ^= 1u;
    }
  } else {
    // ------------------------------------------------------------------ epilogue (kGroups groups share every tile)
    const int g = W4 ? (warp >= 8 ? 1 : 0) : (warp - 4) >> 2;
    const int quad = warp & 3;
    const int row = quad * 32 + lane;
    const uint32_t lane_addr = (uint32_t)(quad * 32) << 16;
    const int et = threadIdx.x & 127;        // 0..127 inside the group (the groups start at multiples of 128)
    volatile int* wflag = wait_flag + 2 * g;
    Ring<2> accring;
    int seg = 0;
    for (int i = pair; i < items; i += args.pairs) {
      const Tile t = tile_at(args, i, row_tiles);
      const int b = accring.s;
      const uint32_t phb = accring.ph;
      accring.advance();
      const int slot = seg & 1;
      ++seg;
      const int n = (2 * t.n2 + (int)rank) * 128 + row;
      const bool n_ok = n < args.N;
      // Scales and destinations of the rows, requested ahead of the sums; two buffers per group: a warp may be one tile ahead of
      // the slowest.
      float* sc = row_scale + (2 * g + slot) * kBN;
      int* to = row_pair + (2 * g + slot) * kBN;
      const float w_scale = n_ok ? args.s1[(size_t)t.expert * args.N + n] : 0.f;
      for (int r = et; r < width(t.rows); r += 128) {
        const bool in = r < t.rows;
        sc[r] = in ? args.ascale[t.row0 + r] : 0.f;
        if (MODE == kOutPairs) to[r] = in ? args.pair_of_pos[t.row0 + r] : 0;
      }
      // One thread of the group performs the bounded wait and publishes the outcome, so that its 128 threads always agree
      // on it (they meet at a named barrier and must never split up).
      if (et == 0) {
        const bool done = ptx::mbar_wait_bounded(bar_accfull + 8 * b, phb, kWaitLimitNs);
        if (!done) atomicExch(args.status, 177);
        wflag[slot] = done ? 1 : 0;
      }
      asm volatile("bar.sync %0, 128;" ::"r"(g + 1) : "memory");
      if (wflag[slot] == 0) break;
      ptx::tc_fence_after();
      const uint32_t acc = tmem_base + b * kBN + lane_addr;
#pragma unroll 1
      for (int c0 = 16 * g; c0 < t.rows; c0 += 16 * C::kGroups) {
        int v[16];
        ptx::tmem_ld16(acc + c0, v);
        ptx::tc_wait_ld();
        store_rows<MODE>(args.epi, v, (long)t.row0 + c0, t.rows - c0, n, n_ok, w_scale, sc + c0, to + c0, 0);
      }
      // this warp's reads of the accumulator are complete: the MMA warp may reuse it
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (rank == 0) ptx::mbar_arrive(bar_accfree + 8 * b);
        else ptx::mbar_arrive_remote(leader_accfree + 8 * b);
      }
    }
  }

  // Both CTAs are done with each other's shared and tensor memory before either releases anything.
  __syncwarp();
  ptx::tc_fence_before();
  __syncthreads();
  ptx::cluster_sync_all();
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc_pair(tmem_base, 512);
  }
}

template <bool W4, int MODE>
static int launch_pair(const Product& p, const Plan& plan, cudaStream_t st) {
  using C = Cfg<W4>;
  auto kern = &experts_pair_kernel<W4, MODE>;
  static std::mutex mu;
  static int most[64] = {};   // CTA pairs that are resident together
  int dev = 0;
  cudaGetDevice(&dev);
  int cap;
  {
    std::lock_guard<std::mutex> lock(mu);
    int& v = most[dev & 63];
    if (v == 0) {
      const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes);
      if (e != cudaSuccess) {
        record_cuda_error(e, "cudaFuncSetAttribute(experts_pair_kernel)");
        return LQ_ERR_CUDA;
      }
      v = sm_count() / 2;
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(2 * v);
      cfg.blockDim = dim3(C::kThreads);
      cfg.dynamicSmemBytes = C::kSmemBytes;
      int clusters = 0;
      if (cudaOccupancyMaxActiveClusters(&clusters, kern, &cfg) == cudaSuccess && clusters > 0 && clusters < v) v = clusters;
      cudaGetLastError();
      if (v < 1) v = 1;
    }
    cap = v;
  }
  Maps maps;
  for (int i = 0; i < C::kBN / 32; ++i)
    if (int rc = make_byte_matrix_map(&maps.x[i], p.x, p.rows, p.K, 16 * (i + 1), 128)) return rc;
  for (int i = C::kBN / 32; i < kPairRowsInt8 / 32; ++i) maps.x[i] = maps.x[0];   // (no width selects these)
  if (W4) maps.w = maps.x[0];
  else if (int rc = make_byte_matrix_map(&maps.w, p.w, (long)p.E * p.N, p.K, 128, 128)) return rc;
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
  a.status = status_word();
  a.N = p.N;
  a.kt_total = p.K / 128;
  a.n_tiles = (p.N + 127) / 128;
  a.n2_tiles = (p.N + 255) / 256;
  if (!a.status) return LQ_ERR_CUDA;
  const long items = max_tiles(p.rows, p.E, plan.bn) * a.n2_tiles;
  a.pairs = (int)(items < cap ? items : cap);
  const cudaError_t e = launch_overlapped(kern, dim3(2 * a.pairs), dim3(C::kThreads), (size_t)C::kSmemBytes, st, maps, a);
  if (e != cudaSuccess) {
    record_cuda_error(e, "experts_pair_kernel launch");
    return LQ_ERR_CUDA;
  }
  return check_launch("experts_pair_kernel");
}

template <bool W4>
static int launch_kind(const Product& p, const Plan& plan, cudaStream_t st) {
  if (p.out_mode == kOutPairs) return launch_pair<W4, kOutPairs>(p, plan, st);
  return launch_pair<W4, kOutGated>(p, plan, st);
}

}  // namespace pair

int run_product_pair(const Product& p, const Plan& plan, cudaStream_t st) {
  if (p.out_mode == kOutPlanes || plan.bn != (p.w_kind == kBlob ? kPairRowsBlob : kPairRowsInt8)) return LQ_ERR_BAD_ARG;
  return p.w_kind == kBlob ? pair::launch_kind<true>(p, plan, st) : pair::launch_kind<false>(p, plan, st);
}

}  // namespace experts
}  // namespace lq
