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
};
// Cuts that give the shortest time: rounds of CTAs times k-steps of a range, with six steps for its start and end.
__host__ __device__ inline int best_splits(long tiles, const SplitRule& r, int slots) {
  int best = 1;
  long least = 0;
  for (int s = 1; s <= r.most; ++s) {
    const long items = tiles * r.n_tiles * s;
    const long cost = (items + slots - 1) / slots * ((r.kt + s - 1) / s + 6);
    if (s == 1 || cost < least) best = s, least = cost;
  }
  return best;
}
struct Plan {
  int* counts;        // [4]: tiles, rows, k-ranges of the first product and of the second
  int4* tiles;        // [max_tiles]
  int* pos_of_pair;   // [pairs]
  int* pair_of_pos;   // [pairs]
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
