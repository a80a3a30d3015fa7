// Epilogue of the grouped products (lq_experts.cu, lq_experts_pair.cu): sixteen sorted rows of one output channel per thread, straight
// from the accumulator.  lane = channel, so that a warp's stores cover 32 neighbouring channels of a row.
#pragma once

#include "lq_experts.cuh"

namespace lq {
namespace experts {

// The 128 codes of a weight row of a blob tile (four 16-byte chunks; step and offset of both groups in `meta`) as INT8, four a word in the
// order of the operand's columns.  (The upper nibbles without a shift, as the upper half of (16 code) * (step << 28): 3 % slower, that
// product has a quarter of the rate.)
__device__ __forceinline__ void unpack_row(const uint4 (&ch)[4], uint32_t meta, uint32_t (&v)[32]) {
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const uint32_t m = c < 2 ? meta : meta >> 16;
    const uint32_t step = m & 0xffu, ab = ((m >> 8) & 0xffu) * 0x01010101u;
    const uint32_t pk[4] = {ch[c].x, ch[c].y, ch[c].z, ch[c].w};
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      v[8 * c + 2 * h] = lqq_dequant4(pk[h] & 0x0F0F0F0Fu, step, ab);
      v[8 * c + 2 * h + 1] = lqq_dequant4((pk[h] >> 4) & 0x0F0F0F0Fu, step, ab);
    }
  }
}

// silu(g) * u.  The hidden values are quantised next, which turns an error of d counts into a wrong code with probability
// d: expf (2 units in the last place) rather than the faster exponential, whose error grows with |g|.  The reciprocal
// is the approximate one: one unit, against half of one and a dozen instructions for the division (in the pair kernel the
// epilogue of a gated tile has to fit beside the unpacking of the next).  exp(-g) = inf gives 0, as the limit does.
__device__ __forceinline__ float gated(float g, float u) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + expf(-g)));
  return __fmul_rn(__fmul_rn(g, r), u);
}

struct EpiArgs {
  void* out;
  unsigned* amax;
  long rows;       // of a plane
  int N, out_dtype;
};

// Scales and destinations of all sixteen rows go to registers first: behind a store the compiler has to fetch them one by one
// (they might be what the store wrote), 130 cycles a row.
template <int DT>
__device__ __forceinline__ void store_pairs(const EpiArgs& a, const int (&v)[16], int valid, int n, float w_scale, const float* sc,
                                            const int* pair) {
  constexpr int ES = DT == LQ_DT_F32 ? 4 : 2;
  float y[16];
  char* at[16];
  char* base = static_cast<char*>(a.out) + (size_t)n * ES;
  const uint32_t pitch = (uint32_t)a.N * ES;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const float4 f = *reinterpret_cast<const float4*>(sc + 4 * q);
    const int4 p = *reinterpret_cast<const int4*>(pair + 4 * q);
    y[4 * q] = lqq_scale(v[4 * q], f.x, w_scale);
    y[4 * q + 1] = lqq_scale(v[4 * q + 1], f.y, w_scale);
    y[4 * q + 2] = lqq_scale(v[4 * q + 2], f.z, w_scale);
    y[4 * q + 3] = lqq_scale(v[4 * q + 3], f.w, w_scale);
    at[4 * q] = base + (uint64_t)pitch * (uint32_t)p.x;
    at[4 * q + 1] = base + (uint64_t)pitch * (uint32_t)p.y;
    at[4 * q + 2] = base + (uint64_t)pitch * (uint32_t)p.z;
    at[4 * q + 3] = base + (uint64_t)pitch * (uint32_t)p.w;
  }
  if (valid >= 16) {
#pragma unroll
    for (int j = 0; j < 16; ++j) store_out(at[j], 0, y[j], DT);
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (j < valid) store_out(at[j], 0, y[j], DT);
  }
}

// v: the sums of rows p0 .. p0 + 15, of which `valid` exist (at least one), for channel n of an expert (n_ok: it exists).
// sc, pair: the rows' scales and destinations, in shared memory, 16-byte aligned; s: the k-range.
template <int MODE>
__device__ __forceinline__ void store_rows(const EpiArgs& a, const int (&v)[16], long p0, int valid, int n, bool n_ok, float w_scale,
                                           const float* sc, const int* pair, int s) {
  if constexpr (MODE == kOutPlanes) {
    if (n_ok) {
      char* o = reinterpret_cast<char*>(static_cast<int32_t*>(a.out) + ((size_t)s * a.rows + p0) * a.N + n);
      const uint32_t pitch = (uint32_t)a.N * 4u;
      if (valid >= 16) {
#pragma unroll
        for (int j = 0; j < 16; ++j) *reinterpret_cast<int32_t*>(o + (uint64_t)pitch * j) = v[j];
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (j < valid) *reinterpret_cast<int32_t*>(o + (uint64_t)pitch * j) = v[j];
      }
    }
  } else if constexpr (MODE == kOutPairs) {
    if (n_ok) {
      if (a.out_dtype == LQ_DT_BF16) store_pairs<LQ_DT_BF16>(a, v, valid, n, w_scale, sc, pair);
      else if (a.out_dtype == LQ_DT_F16) store_pairs<LQ_DT_F16>(a, v, valid, n, w_scale, sc, pair);
      else store_pairs<LQ_DT_F32>(a, v, valid, n, w_scale, sc, pair);
    }
  } else {
    // An even lane holds the gate and the odd one beside it the up value of the same hidden channel.  The even lane takes rows
    // 0..7 and the odd one rows 8..15, each handing over what the other needs.
    const int lane = threadIdx.x & 31;
    const bool odd = lane & 1;
    const int first = odd ? 8 : 0;
    float h[8];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const float4 lo4 = *reinterpret_cast<const float4*>(sc + 4 * q), hi4 = *reinterpret_cast<const float4*>(sc + 8 + 4 * q);
      const float slo[4] = {lo4.x, lo4.y, lo4.z, lo4.w}, shi[4] = {hi4.x, hi4.y, hi4.z, hi4.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float lo = lqq_scale(v[4 * q + k], slo[k], w_scale), hi = lqq_scale(v[8 + 4 * q + k], shi[k], w_scale);
        const float other = __shfl_xor_sync(0xffffffffu, odd ? lo : hi, 1), own = odd ? hi : lo;
        h[4 * q + k] = gated(odd ? other : own, odd ? own : other);
      }
    }
    const uint32_t pitch = (uint32_t)(a.N / 2) * 4u;
    char* o = reinterpret_cast<char*>(static_cast<float*>(a.out) + (size_t)(p0 + first) * (a.N / 2) + (n >> 1));
    if (valid >= 16) {
#pragma unroll
      for (int j = 0; j < 8; ++j) *reinterpret_cast<float*>(o + (uint64_t)pitch * j) = h[j];
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (first + j < valid) *reinterpret_cast<float*>(o + (uint64_t)pitch * j) = h[j];
    }
    // the rows' largest magnitudes over the warp's 16 hidden channels: after three halving steps every lane holds one row
    float m[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) m[j] = fmaxf(fabsf(h[j]), 0.f);   // a NaN counts as zero, as in the row quantisers
#pragma unroll
    for (int w = 4; w >= 1; w >>= 1) {
      const bool up = lane & (8 / w);   // lane bits 1, 2, 3
#pragma unroll
      for (int j = 0; j < w; ++j) {
        const float keep = up ? m[j + w] : m[j], give = up ? m[j] : m[j + w];
        m[j] = fmaxf(keep, __shfl_xor_sync(0xffffffffu, give, 8 / w));
      }
    }
    m[0] = fmaxf(m[0], __shfl_xor_sync(0xffffffffu, m[0], 16));
    const int row = first + ((lane & 2) ? 4 : 0) + ((lane & 4) ? 2 : 0) + ((lane & 8) ? 1 : 0);
    // magnitudes compare like their bits; the order of the atomics does not matter to a maximum
    if (lane < 16 && row < valid) atomicMax(a.amax + p0 + row, __float_as_uint(m[0]));
  }
}

}  // namespace experts
}  // namespace lq
