// What the kernels of the mixture-of-experts path share: the plan that sorts (token, expert) pairs by expert, and the
// grouped product over it.
#pragma once

#include <stdint.h>

#include "lq_common.cuh"

namespace lq {
namespace experts {

constexpr int kMaxExperts = 512;
constexpr int kMaxTopk = 32;

// Weights of a grouped product: tile blobs of the 4-bit weights, one behind the other, or INT8 rows [E * N, K].
enum WeightKind { kBlob = 0, kInt8 = 1 };

// A stable counting sort of the T * topk pairs by expert: pair i (token i / topk) gets row pos_of_pair[i] of the sorted
// activations, the pair at row p is pair_of_pos[p].  Pairs whose id is no expert get no row (-1).  The rows of an expert
// are cut into tiles of at most `bn` rows; tiles[i] = (expert, first row, rows, 0).
//
// Where few tiles meet many CTA slots a product's k is cut into ranges, whose int32 sums go to planes.  Whether it may be cut is
// decided by the host from the sizes (`most` > 1), how often on the device from the number of tiles the tokens made.
struct SplitRule {
  int n_tiles, kt;   // 128-channel blocks of an expert, k-steps
  int most;          // planes there is room for; 1: k stays whole
  bool even;         // k whole: the k-steps of all tiles may be dealt out evenly (see cut_evenly)
};
// Time of `s` ranges: rounds of CTAs times k-steps of a range, with six steps for its start and end.  Tiles times ranges fit 32 bits where
// a product may be cut (the device divides 32 bits several times as fast as 64, and the product waits).
__host__ __device__ inline unsigned split_cost(unsigned tiles, const SplitRule& r, int s, int slots) {
  return (tiles * r.n_tiles * s + slots - 1) / slots * ((unsigned)(r.kt + s - 1) / s + 6);
}
// With k whole the CTAs' last round is seldom full.  Where that costs more than joining parts of tiles the k-steps of all tiles are
// dealt out in equal, contiguous shares.  A share is a whole tile at least (more tiles than CTAs), so a tile has two parts at most.
// The empty part of the last round counts half, a CTA alone on its SM being nearly twice as fast; against it stand the joins and
// the order in which shares read memory, which cost more the more rounds there are.  Measured, one token, 4096 -> 28672, whole /
// dealt out, us: 2 experts (1.5 rounds of CTAs) 29.3 / 27.2, 3 (2.3) 39.6 / 36.9, 4 (3.0) 46.0 / 45.7, 6 (4.5) 64.6 / 63.8, 8 (6.1) 79.2 /
// 81.2; 8192 -> 28672: 50.5 / 45.2, 70.5 / 62.9, 85.0 / 79.8, 118.9 / 115.0, 150.7 / 149.6; 2048 -> 28672: 19.2 / 18.3, 23.9 / 23.8, 26.5 /
// 28.0, 37.0 / 38.5, 44.1 / 47.3.  With INT8 weights, where the copies are all there is to do, 5 % slower.
constexpr int kEvenRows = 32;    // for plans of this width, with 4-bit weights
__host__ __device__ inline bool cut_evenly(long tiles, const SplitRule& r, int slots) {
  const long items = tiles * r.n_tiles;
  if (items <= slots || items > 8L * slots) return false;
  const unsigned n = (unsigned)items, g = (unsigned)slots, rounds = (n + g - 1) / g;
  return rounds * r.kt > (n * r.kt + g - 1) / g + 4 + 5 * rounds;
}
struct Plan {
  int* counts;        // [4]: tiles, rows, k-ranges of the first product and of the second (0: dealt out evenly)
  int4* tiles;        // [max_tiles]
  int* pos_of_pair;   // [pairs]
  int* pair_of_pos;   // [pairs]
  int4* join[2];      // [slots], zero before each product: for each epilogue warp, parts that are there of the tile cut between two CTAs
  int32_t* part;      // [slots][2][bn][128]: their sums
  int bn, slots;      // slots: CTAs of the tile kernel that run together
  SplitRule rule[2];
};
inline long max_tiles(long pairs, int E, int bn) {
  const long by_rows = pairs / bn + E;
  return by_rows < pairs ? by_rows : pairs;
}

// Outputs of a grouped product, for the sorted row p and output channel n of its expert:
enum OutMode {
  kOutPlanes = 0,   // int32 sums out[s][p][n] of k-range s
  kOutPairs = 1,    // scaled, in `out_dtype`, out[pair_of_pos[p]][n]
  kOutGated = 2     // channels 2c, 2c + 1 = gate, up of hidden channel c: out[p][c] = silu(gate) * up in float32, and the
                    // largest magnitude of each row as the bits of a float in amax[p] (zero before)
};
struct Product {
  const void* w;
  int w_kind;
  const float* s1;         // [E, N]
  const int8_t* x;         // [rows, K], sorted
  const float* ascale;     // [rows]
  long rows;               // rows of `x`: at least as many as the plan has
  int E, N, K;
  int which;               // of the plan's rules (kOutPlanes; k is whole otherwise)
  int out_mode, out_dtype;
  void* out;
  unsigned* amax;
};
int run_product(const Product& p, const Plan& plan, cudaStream_t st);        // lq_experts.cu
// Tiles of the CTA-pair kernel (lq_experts_pair.cu), which run_product takes for plans of that width.
constexpr int kPairRowsBlob = 192, kPairRowsInt8 = 256;
int run_product_pair(const Product& p, const Plan& plan, cudaStream_t st);

}  // namespace experts
}  // namespace lq
