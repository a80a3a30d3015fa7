// Norms around a block: the norm of the block's output, gate, scales, residual and the norm before the next block in one
// pass over the rows, to 16- / 32-bit rows or to the INT8 rows and scales that the linears read.
#include <type_traits>

#include "lq_common.cuh"

namespace lq {

// Row m of an operand lies at base + (m / inner) * outer_stride + (m % inner) * inner_stride elements.
struct RowStrides {
  long outer, inner;
};

struct NormArgs {
  const void* x;
  const void* residual;
  const void* gate;
  const void* weight;
  const void* post;
  void* z;         // rows of x's type, or
  int8_t* q;       // INT8 rows with
  float* q_scale;  // one scale each
  void* h;         // the stream (null: not stored)
  RowStrides xs, rs, gs;
  int gate_step;   // 1, or 0: one gate for a row
  int rows, inner, H;
  double inv_h, eps, scale, residual_scale;
  float offset;
  bool weight_f32, post_f32, gate_f32;   // float32 instead of x's type
};

// A unit: eight elements of a thread, neighbours (VEC; 16-byte accesses) or 32 apart, so that a warp has 256 neighbours.
template <bool VEC>
__device__ __forceinline__ int unit_at(int i) {
  return VEC ? (i * blockDim.x + threadIdx.x) * 8 : ((i * (blockDim.x >> 5) + (threadIdx.x >> 5)) * 256) + (threadIdx.x & 31);
}

template <typename T, bool VEC>
struct Eight {
  uint4 raw[sizeof(T) / 2];
  // Elements that a pass reads once; KEEP: by all rows, so that they stay in L1.
  template <bool KEEP = false>
  __device__ __forceinline__ void load(const T* p, int at, int H) {
#pragma unroll
    for (int w = 0; w < (int)sizeof(T) / 2; ++w) {
      raw[w] = make_uint4(0u, 0u, 0u, 0u);
      if (at < H) raw[w] = KEEP ? *reinterpret_cast<const uint4*>(p + at + w * 4) : ld_stream_v4(p + at + w * 4);
    }
  }
  __device__ __forceinline__ void floats(float2 (&v)[4]) const {
    if constexpr (sizeof(T) == 2) {
      vec_floats<T>(raw[0], v);
    } else {
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        v[2 * w] = make_float2(__uint_as_float(raw[w].x), __uint_as_float(raw[w].y));
        v[2 * w + 1] = make_float2(__uint_as_float(raw[w].z), __uint_as_float(raw[w].w));
      }
    }
  }
};
template <typename T>
struct Eight<T, false> {
  float2 f[4];
  template <bool KEEP = false>
  __device__ __forceinline__ void load(const T* p, int at, int H) {
    p += at;
    T e[8];
    if (at + 7 * 32 < H) {
#pragma unroll
      for (int j = 0; j < 8; ++j) e[j] = p[j * 32];
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) e[j] = at + j * 32 < H ? p[j * 32] : T(0.f);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = make_float2(to_f32<T>(e[2 * j]), to_f32<T>(e[2 * j + 1]));
  }
  __device__ __forceinline__ void floats(float2 (&v)[4]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = f[j];
  }
};

__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tmul.rn.f32x2 rd, ra, rb;\n\t"
      "mov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// A vector in x's type or in float32, plus `offset`.
template <typename T, bool VEC>
__device__ __forceinline__ void load_weight(const void* p, bool f32, float offset, int at, int H, float2 (&v)[4]) {
  if (f32) {
    Eight<float, VEC> e;
    e.template load<true>(static_cast<const float*>(p), at, H);
    e.floats(v);
  } else {
    Eight<T, VEC> e;
    e.template load<true>(static_cast<const T*>(p), at, H);
    e.floats(v);
  }
  if (offset != 0.f)
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = add2(v[j], both(offset));
}

// Two numbers rounded to T, as they lie in memory (16-bit types).
template <typename T> __device__ __forceinline__ uint32_t pack2(float2 v);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float2 v) {
  const __half2 h = __float22half2_rn(v);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float2 v) {
  const __nv_bfloat162 h = __float22bfloat162_rn(v);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Eight numbers rounded to T: what is stored, and what that stands for.
template <typename T>
struct Rounded {
  uint32_t w[8 * sizeof(T) / 4];
  __device__ __forceinline__ Rounded(const float2 (&v)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (sizeof(T) == 2) w[j] = pack2<T>(v[j]);
      else w[2 * j] = __float_as_uint(v[j].x), w[2 * j + 1] = __float_as_uint(v[j].y);
    }
  }
  __device__ __forceinline__ void floats(float2 (&v)[4]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (sizeof(T) == 2) v[j] = unpack2<T>(w[j]);
    }
  }
  template <bool VEC>
  __device__ __forceinline__ void store(T* p, int at, int H) const {
    if constexpr (VEC) {
      if (at >= H) return;
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i)
        reinterpret_cast<uint4*>(p + at)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    } else {
      using Bits = std::conditional_t<sizeof(T) == 2, uint16_t, uint32_t>;
      Bits* to = reinterpret_cast<Bits*>(p) + at;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (at + j * 32 < H) to[j * 32] = (Bits)(sizeof(T) == 2 ? w[j / 2] >> (16 * (j & 1)) : w[sizeof(T) == 2 ? 0 : j]);
    }
  }
};

// Sum, and maximum of numbers that are not negative (a NaN counts as more than all others), over the CTA: the same bits in
// every thread.  `red`: 64 floats, 16-byte aligned, that nobody has read since the last barrier; 0 where there is no warp.
template <bool MAX>
__device__ __forceinline__ float2 block_sum_max(float s, float m, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (MAX) m = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(m)));
  const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  if ((threadIdx.x & 31) == 0) {
    red[warp] = s;
    if (MAX) red[32 + warp] = m;
  }
  __syncthreads();
  s = 0.f, m = 0.f;
  for (int w = 0; w < warps; w += 4) {   // (read by all at once: broadcasts)
    const float4 p = *reinterpret_cast<const float4*>(red + w);
    s += (p.x + p.y) + (p.z + p.w);
    if (MAX) {
      const uint4 q = *reinterpret_cast<const uint4*>(red + 32 + w);
      m = __uint_as_float(max(max(__float_as_uint(m), max(q.x, q.y)), max(q.z, q.w)));
    }
  }
  return make_float2(s, m);
}

// A factor of a whole row as the float32 number next to it on the side of zero and what that leaves of it.  The rest is never quite 0 (beside a
// factor that dwarfs it: 2^-49), so that both take an infinity to the same one; factors smaller than that are what they are, 0 among them.
struct Factor {
  float hi, lo;
};
__device__ __forceinline__ Factor split(double f) {
  const float hi = __double2float_rz(f);
  const float lo = fabsf(hi) < INFINITY ? (float)(f - (double)hi) : 0.f;
  return {hi, lo == 0.f && fabsf(hi) >= 0x1p-100f ? copysignf(0x1p-149f, hi) : lo};
}

// (mean of squares + eps)^-1/2 in 64 bits: a float32 root and one step of Newton's iteration.
__device__ __forceinline__ double exact_root(float ss, const NormArgs& a) {
  const double m = (double)ss * a.inv_h + a.eps;
  const float r = rsqrtf((float)m);
  return r < INFINITY ? fma(0.5 * r, fma(-m * r, (double)r, 1.0), (double)r) : (double)r;
}

// round(127 t / top) of an element that lies next to a border between two codes, or whose factor 127 / top float32 does not
// hold.  The product by 127 is exact and the quotient of two float32 numbers is never nearer to a half-integer than 64 bits can
// tell, unless it is one.
__device__ __noinline__ int code_exact(float t, float top) {
  const double q = 127.0 * (double)t / (double)top;
  return q == q ? max(-127, min(127, __double2int_rn(q))) : 0;
}

template <typename T> __device__ __forceinline__ T rounded(double v);
template <> __device__ __forceinline__ float rounded<float>(double v) { return (float)v; }
template <> __device__ __forceinline__ __half rounded<__half>(double v) { return __float2half_rn((float)v); }
template <> __device__ __forceinline__ __nv_bfloat16 rounded<__nv_bfloat16>(double v) { return __float2bfloat16_rn((float)v); }

__device__ __forceinline__ long row_start(const RowStrides& s, unsigned m, const NormArgs& a) {
  if (a.inner == a.rows) return (long)m * s.inner;
  const unsigned outer = m / (unsigned)a.inner;
  return (long)outer * s.outer + (long)(m - outer * a.inner) * s.inner;
}

// Whether float32 holds a row's sum of squares, and the `mean` of them and eps: each square may be off by 2^-150, 2^-30 of the least mean here.
__device__ __forceinline__ bool holds(float ss, float mean) { return ss < 3e38f && mean >= 0x1p-120f; }

// A row of which it does not, element by element in 64 bits: from its operands in memory, or, where that is `formed` for good, from its
// stream.  A function of its own that ends the row: what hardly any row takes then costs the others no registers (the elements taken again
// inside the kernel's own code: 7 to 24 % of all rows' time where 16-byte accesses do not go).  Batches of nothing else take two to six
// times as long (4096 x 4096 to INT8 92 us, 144 with a post-norm).  `sums`: 32 doubles, the maxima behind them.
template <typename T, typename R, bool QUANT>
__device__ __noinline__ void outlying_row(const NormArgs& a, unsigned m, bool formed, double* sums) {
  const int H = a.H, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  float* tops = reinterpret_cast<float*>(sums + 32);
  auto sum_max = [&](double s, float& top) {
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
    __syncthreads();   // (what was read from there before)
    if ((threadIdx.x & 31) == 0) sums[warp] = s, tops[warp] = top;
    __syncthreads();
    s = 0.0;
    for (int w = 0; w < warps; ++w) s += sums[w], top = __uint_as_float(max(__float_as_uint(top), __float_as_uint(tops[w])));
    return s;
  };
  auto weight = [&](const void* p, bool f32, int e) {
    return (f32 ? static_cast<const float*>(p)[e] : to_f32<T>(static_cast<const T*>(p)[e])) + a.offset;
  };
  auto root_of = [&](double s) { return s == 0.0 ? 0.0 : rsqrt(s * a.inv_h + a.eps); };   // (zeros stay zeros, whatever eps)
  const T* x = static_cast<const T*>(a.x) + row_start(a.xs, m, a);
  R* h = static_cast<R*>(a.h) + (long)m * H;
  const R* row = a.h ? h : reinterpret_cast<const R*>(x);
  double s = 0.0, root = 1.0;
  float top = 0.f;
  __syncthreads();   // (the stream as the other threads stored it)
  if (a.post && !formed) {
#pragma unroll 1
    for (int e = threadIdx.x; e < H; e += blockDim.x) s = fma((double)to_f32<T>(x[e]), (double)to_f32<T>(x[e]), s);
    root = root_of(sum_max(s, top));
  }
  s = 0.0;
#pragma unroll 1
  for (int e = threadIdx.x; e < H; e += blockDim.x) {
    if (!formed) {
      double p = a.scale * root * to_f32<T>(x[e]);
      if (a.post) p *= weight(a.post, a.post_f32, e);
      if (a.gate) {
        const long at = row_start(a.gs, m, a) + (a.gate_step ? e : 0);
        p *= a.gate_f32 ? static_cast<const float*>(a.gate)[at] : to_f32<T>(static_cast<const T*>(a.gate)[at]);
      }
      if (a.residual) p = fma(a.residual_scale, (double)to_f32<R>((static_cast<const R*>(a.residual) + row_start(a.rs, m, a))[e]), p);
      h[e] = rounded<R>(p);
    }
    const float v = to_f32<R>(row[e]), t = a.weight ? v * weight(a.weight, a.weight_f32, e) : v;
    s = fma((double)v, (double)v, s);
    top = max_abs_nan(top, t, t);
  }
  root = root_of(sum_max(s, top));
  if (QUANT && threadIdx.x == 0) a.q_scale[m] = (float)(top * root / 127.0);
#pragma unroll 1
  for (int e = threadIdx.x; e < H; e += blockDim.x) {
    const float v = to_f32<R>(row[e]), w = a.weight ? weight(a.weight, a.weight_f32, e) : 1.f;
    if constexpr (QUANT) a.q[(long)m * H + e] = (int8_t)code_exact(v * w, top);
    else static_cast<T*>(a.z)[(long)m * H + e] = rounded<T>(v * root * w);
  }
}

// A CTA takes row after row, each in registers (NV units of eight elements a thread), so that everything is read once:
//   p = x * (mean(x^2) + eps)^-1/2 * (post + offset)        (with `post`; x otherwise)
//   h = residual_scale * residual + scale * gate * p         rounded to the stream's type R, and stored
//   z = h * (mean(h^2) + eps)^-1/2 * (weight + offset)       of the rounded h
// in float32.  QUANT: INT8 rows instead of z.  The root is the same for a whole row, so it cancels out of
// codes = round(127 z / max|z|): with t = h * (weight + offset) they are round(127 t / max|t|), exactly (t is a float32
// product, exact where both factors have 16 bits), and the root goes into the row's scale alone, max|t| * root / 127: one reduction for
// the sum and the maximum, and codes that do not hang on the order of a sum.
// Elements are multiplied by their own factors first (exact for 16-bit types) and by the row's factors (roots and scales, in 64
// bits, as two float32 numbers) last: h then hangs on two roundings only before its own, and half as many elements as in the
// order of the formula fall on the other side of a border between two 16-bit numbers than in 64 bits.
// Bound by the chain of launch, load, reduction(s) and store at few rows (one of 4096: 2.6 us, a launch takes 2.2), by memory at
// many (16384 x 8192 bf16, stream added and stored: 184 us, 5.8 TB/s; with a float32 stream and gates 310 us, 6.1), and by instruction
// issue where the rows are quantised as well (4096 x 4096: 25 us, 4.6 TB/s), spilled registers among it: 64 a thread, which let an
// SM hold 1024 threads, do not take all that a row carries (stack bytes a thread at one, two and four units: 0, 8 to 48 and 112 to 272 to
// 16- and 32-bit rows, 24 to 48, 56 to 120 and 184 to 344 to INT8; single elements at two, four and eight: 56 to 128, 256 to 320, 648 to 744).
// Vectors that all rows share stay in L1.  Measured beside it: rows asked for ahead, into registers (fewer warps: 10 to 40 % slower) or through a ring in shared memory (cp.async, two and three
// rows; 170 us for the first of these, 5 to 15 % slower elsewhere); four units a thread on 128 threads (25 us for the last, but 89 instead
// of 58 at 4096 x 8192).  Rows that 16-byte accesses cannot take (8192 x 5001: 109 us, 3.0 TB/s) are bound by instruction issue too.
template <typename T, typename R, int NV, bool VEC, bool QUANT>
__global__ void __launch_bounds__(VEC ? 1024 : 512, VEC ? 1 : 2)
block_norm_kernel(const __grid_constant__ NormArgs a) {
  __shared__ __align__(16) float red[2][2][64];
  __shared__ double outlying[48];
  constexpr bool HOLD = VEC && NV == 1 && !QUANT;
  for (int i = threadIdx.x; i < 2 * 2 * 64; i += blockDim.x) (&red[0][0][0])[i] = 0.f;
  __syncthreads();
  allow_dependents();
  dependency_wait();
  const int H = a.H;
  const bool gate16 = a.gate && a.gate_step && !a.gate_f32;
  auto row_at = [&](const RowStrides& s, unsigned m) { return row_start(s, m, a); };
  const Factor rs = split(a.residual_scale);
  const bool sum = a.residual && !a.post && a.scale == 1.0 && a.residual_scale == 1.0;   // h = residual + gate * x
  const Factor scale = split(a.scale);
  const float inv_h = (float)a.inv_h, eps = (float)a.eps;
  int parity = 0;
  for (unsigned m = blockIdx.x; m < (unsigned)a.rows; m += gridDim.x, parity ^= 1) {
    const T* x = static_cast<const T*>(a.x) + row_at(a.xs, m);
    Eight<T, VEC> rx[NV], rg[NV];
    Eight<R, VEC> rr[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) rx[i].load(x, unit_at<VEC>(i), H);
    if (a.residual) {
      const R* r = static_cast<const R*>(a.residual) + row_at(a.rs, m);
#pragma unroll
      for (int i = 0; i < NV; ++i) rr[i].load(r, unit_at<VEC>(i), H);
    }
    if (gate16) {
      const T* g = static_cast<const T*>(a.gate) + row_at(a.gs, m);
#pragma unroll
      for (int i = 0; i < NV; ++i) rg[i].load(g, unit_at<VEC>(i), H);
    }
    float2 v[NV][4];
#pragma unroll
    for (int i = 0; i < NV; ++i) rx[i].floats(v[i]);
    float row_gate = 1.f;
    if (a.gate && !a.gate_step) {
      const long at = row_at(a.gs, m);
      row_gate = a.gate_f32 ? static_cast<const float*>(a.gate)[at] : to_f32<T>(static_cast<const T*>(a.gate)[at]);
    }
    Factor by = scale;
    if (a.post) {
      float2 s = both(0.f);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float2 w[4];
        load_weight<T, VEC>(a.post, a.post_f32, a.offset, unit_at<VEC>(i), H, w);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          s = fma2(v[i][j], v[i][j], s);
          v[i][j] = mul2(v[i][j], w[j]);
        }
      }
      // (every thread takes the same way: the sum has the same bits everywhere)
      const float ss = block_sum_max<false>(s.x + s.y, 0.f, red[parity][0]).x;
      if (!holds(ss, __fmaf_rn(ss, inv_h, eps))) {   // (float32 may not hold the elements times a weight and a gate either)
        outlying_row<T, R, QUANT>(a, m, false, outlying);
        continue;
      }
      by = split(exact_root(ss, a) * a.scale);
    }
    if (a.gate) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float2 g[4] = {both(row_gate), both(row_gate), both(row_gate), both(row_gate)};
        if (gate16) rg[i].floats(g);
        else if (a.gate_step) {
          Eight<float, VEC> e;
          e.load(static_cast<const float*>(a.gate) + row_at(a.gs, m), unit_at<VEC>(i), H);
          e.floats(g);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) v[i][j] = mul2(v[i][j], g[j]);
      }
    }
    // the stream: formed and rounded in place of x
    R* row = static_cast<R*>(a.h) + (long)m * H;
    float2 ss2 = both(0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (a.h) {   // (nothing joins otherwise: x stays as it is)
        float2 u[4];
        if (a.residual) {
          rr[i].floats(u);
          if (sum) {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[i][j] = add2(v[i][j], u[j]);
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              v[i][j] = fma2(u[j], both(rs.hi), fma2(v[i][j], both(by.hi), fma2(v[i][j], both(by.lo), mul2(u[j], both(rs.lo)))));
          }
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) v[i][j] = fma2(v[i][j], both(by.hi), mul2(v[i][j], both(by.lo)));
        }
        const Rounded<R> h(v[i]);
        h.floats(v[i]);
        h.template store<VEC>(row, unit_at<VEC>(i), H);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) ss2 = fma2(v[i][j], v[i][j], ss2);
    }
    float2 w[HOLD ? NV : 1][4];   // the norm's weight, held where there are registers for it
    float top = 0.f;
    if constexpr (QUANT || HOLD) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float2 (&wi)[4] = w[HOLD ? i : 0];
        if (a.weight) load_weight<T, VEC>(a.weight, a.weight_f32, a.offset, unit_at<VEC>(i), H, wi);
        if constexpr (QUANT) {   // v: the rows times the weight
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (a.weight) v[i][j] = mul2(v[i][j], wi[j]);
            top = max_abs_nan(top, v[i][j].x, v[i][j].y);
          }
        }
      }
    }
    const float2 both_of = block_sum_max<QUANT>(ss2.x + ss2.y, top, red[parity][1]);
    const float mean = __fmaf_rn(both_of.x, inv_h, eps);
    if (!holds(both_of.x, mean)) {
      // (from the operands again: a product with the gate that float32 did not hold may have made it so; not where h took the place of one)
      outlying_row<T, R, QUANT>(a, m, !a.h || a.h == a.x || a.h == a.residual, outlying);
      continue;
    }
    float root = 0.f;
    if (!QUANT || threadIdx.x == 0) root = __frsqrt_rn(mean);
    if constexpr (!QUANT) {
      T* z = static_cast<T*>(a.z) + (long)m * H;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float2 (&wi)[4] = w[HOLD ? i : 0];
        if (!HOLD && a.weight) load_weight<T, VEC>(a.weight, a.weight_f32, a.offset, unit_at<VEC>(i), H, wi);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (a.weight) v[i][j] = mul2(v[i][j], wi[j]);
          v[i][j] = mul2(v[i][j], both(root));
        }
        Rounded<T>(v[i]).template store<VEC>(z, unit_at<VEC>(i), H);
      }
    } else {
      top = both_of.y;
      if (threadIdx.x == 0) a.q_scale[m] = __fdiv_rn(top * root, 127.0f);
      const float inv = __fdiv_rn(127.0f, top);
      int8_t* q = a.q + (long)m * H;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float2 r[4];
        const bool safe = inv < 3e38f && round_quotients(v[i], inv, r);
        uint32_t c[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) c[2 * j] = __float_as_uint(r[j].x), c[2 * j + 1] = __float_as_uint(r[j].y);
        if (!safe) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float t = j & 1 ? v[i][j / 2].y : v[i][j / 2].x;
            if (!(inv < 3e38f) || !near_integer(t, inv)) c[j] = (uint32_t)code_exact(t, top);
          }
        }
        const int at = unit_at<VEC>(i);
        if constexpr (VEC) {
          if (at < H)
            *reinterpret_cast<uint2*>(q + at) =
                make_uint2(__byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410),
                           __byte_perm(__byte_perm(c[4], c[5], 0x0040), __byte_perm(c[6], c[7], 0x0040), 0x5410));
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (at + j * 32 < H) q[at + j * 32] = (int8_t)c[j];
        }
      }
    }
  }
}

// As many CTAs as the GPU holds at once (64 registers a thread), or fewer where all of them then take as many rows.
template <typename K>
static cudaError_t launch_rows(K* kernel, const NormArgs& a, int threads, cudaStream_t st) {
  const long most = 1024 / threads * sm_count(), turns = (a.rows + most - 1) / most;
  return launch_overlapped(kernel, dim3((unsigned)((a.rows + turns - 1) / turns)), dim3(threads), 0, st, a);
}

template <typename T, typename R, int NV, bool QUANT>
static cudaError_t launch_norm(const NormArgs& a, int threads, bool vec, cudaStream_t st) {
  if constexpr (NV <= 4)
    if (vec) return launch_rows(block_norm_kernel<T, R, NV, true, QUANT>, a, threads, st);
  if constexpr (NV >= 2) return launch_rows(block_norm_kernel<T, R, NV, false, QUANT>, a, threads, st);
  return cudaErrorInvalidValue;   // (none: launch_norm_nv takes NV 1 for 16-byte accesses, NV 8 for single elements alone)
}

template <typename T, typename R, int NV>
static cudaError_t launch_norm_q(const NormArgs& a, int threads, bool vec, cudaStream_t st) {
  return a.q ? launch_norm<T, R, NV, true>(a, threads, vec, st) : launch_norm<T, R, NV, false>(a, threads, vec, st);
}

// Rows that the GPU holds all at once are spread wide (their time is a chain of latencies); of many, a thread takes two units of each, so
// that the fixed work of a warp for a row (its reductions) is shared by more elements.
template <typename T, typename R>
static cudaError_t launch_norm_nv(const NormArgs& a, bool vec, cudaStream_t st) {
  const int units = vec ? (a.H + 7) / 8 : (a.H + 255) / 256 * 32;
  auto threads = [&](int nv) { return (units + nv * 32 - 1) / (nv * 32) * 32; };
  if (!vec) {
    if (threads(2) <= 512) return launch_norm_q<T, R, 2>(a, threads(2), vec, st);
    return threads(4) <= 512 ? launch_norm_q<T, R, 4>(a, threads(4), vec, st) : launch_norm_q<T, R, 8>(a, threads(8), vec, st);
  }
  if (threads(1) <= 1024 && (long)a.rows * threads(1) <= (long)sm_count() * 1024) return launch_norm_q<T, R, 1>(a, threads(1), vec, st);
  if (threads(2) <= 1024) return launch_norm_q<T, R, 2>(a, threads(2), vec, st);
  return launch_norm_q<T, R, 4>(a, threads(4), vec, st);
}

}  // namespace lq

extern "C" int lq_block_norm(const void* x, int x_dtype, long x_outer, long x_inner, const void* residual, int stream_dtype,
                             long r_outer, long r_inner, const void* gate, int gate_dtype, long g_outer, long g_inner,
                             int gate_step, const void* weight, int weight_dtype, const void* post, int post_dtype, void* z,
                             int8_t* q, float* q_scale, void* h, int rows, int inner, int H, double eps, double scale,
                             double residual_scale, double offset, void* stream) {
  using namespace lq;
  if (!x || rows <= 0 || inner <= 0 || H <= 0 || x_dtype < 0 || x_dtype > 2 || (z == nullptr) == (q == nullptr) ||
      (q != nullptr) != (q_scale != nullptr))
    return LQ_ERR_BAD_ARG;
  if (stream_dtype != x_dtype && !(residual && stream_dtype == LQ_DT_F32)) return LQ_ERR_BAD_ARG;
  const int side[3][2] = {{gate != nullptr, gate_dtype}, {weight != nullptr, weight_dtype}, {post != nullptr, post_dtype}};
  for (const auto& s : side)
    if (s[0] && s[1] != x_dtype && s[1] != LQ_DT_F32) return LQ_ERR_BAD_ARG;
  if (gate && gate_step != 0 && gate_step != 1) return LQ_ERR_BAD_ARG;
  if (!(eps >= 0.0)) return LQ_ERR_BAD_ARG;
  if (!h && (residual || gate || post || scale != 1.0)) return LQ_ERR_BAD_ARG;
  if (H > 32768) return LQ_ERR_SHAPE;
  NormArgs a = {};
  a.x = x, a.residual = residual, a.gate = gate, a.weight = weight, a.post = post;
  a.z = z, a.q = q, a.q_scale = q_scale, a.h = h;
  a.xs = {x_outer, x_inner}, a.rs = {r_outer, r_inner}, a.gs = {g_outer, g_inner};
  a.gate_step = gate_step, a.rows = rows, a.inner = inner, a.H = H;
  a.inv_h = 1.0 / H, a.eps = eps, a.scale = scale, a.residual_scale = residual_scale, a.offset = (float)offset;
  a.weight_f32 = weight_dtype == LQ_DT_F32, a.post_f32 = post_dtype == LQ_DT_F32, a.gate_f32 = gate_dtype == LQ_DT_F32;
  // 16-byte accesses everywhere, or single elements everywhere
  auto odd = [](const void* p, int dtype, long s0, long s1) {
    const long size = dtype == LQ_DT_F32 ? 4 : 2;
    return p && ((reinterpret_cast<uintptr_t>(p) | (uintptr_t)(s0 * size) | (uintptr_t)(s1 * size)) & 15) != 0;
  };
  const bool vec = H % 8 == 0 && !odd(x, x_dtype, x_outer, x_inner) && !odd(residual, stream_dtype, r_outer, r_inner) &&
                   !(gate && gate_step && odd(gate, gate_dtype, g_outer, g_inner)) && !odd(weight, weight_dtype, 0, 0) &&
                   !odd(post, post_dtype, 0, 0) && !odd(z, x_dtype, 0, 0) && !odd(h, stream_dtype, 0, 0) &&
                   (reinterpret_cast<uintptr_t>(q) & 7) == 0;
  cudaStream_t st = as_stream(stream);
  cudaError_t e;
  if (x_dtype == LQ_DT_F32) e = launch_norm_nv<float, float>(a, vec, st);
  else if (x_dtype == LQ_DT_BF16)
    e = stream_dtype == LQ_DT_F32 ? launch_norm_nv<__nv_bfloat16, float>(a, vec, st)
                                  : launch_norm_nv<__nv_bfloat16, __nv_bfloat16>(a, vec, st);
  else
    e = stream_dtype == LQ_DT_F32 ? launch_norm_nv<__half, float>(a, vec, st)
                                  : launch_norm_nv<__half, __half>(a, vec, st);
  if (e != cudaSuccess) {
    record_cuda_error(e, "block_norm_kernel");
    return LQ_ERR_CUDA;
  }
  return check_launch("block_norm_kernel");
}
