// Norms around a block: the norm of the block's output, gate, scales, residual and the norm before the next block in one
// pass over the rows, to 16- / 32-bit rows or to the INT8 rows and scales that the linears read.
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
  int inner, H;
  float eps, scale, residual_scale, offset;
  bool weight_f32, post_f32, gate_f32;   // float32 instead of x's type
};

// Eight elements of a thread: neighbours (VEC; 16-byte accesses), or `blockDim.x` apart.
template <bool VEC>
__device__ __forceinline__ int unit_at(int i) {
  return VEC ? (i * blockDim.x + threadIdx.x) * 8 : i * blockDim.x * 8 + threadIdx.x;
}

template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, int at, int H, float (&v)[8]) {
  if constexpr (VEC) {
    if (at < H) {
      constexpr int W = sizeof(T) / 2;
      float2 f[4];
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const uint4 raw = ld_stream_v4(p + at + w * 4);
        if constexpr (W == 1) vec_floats<T>(raw, f);
        else {
          f[2 * w] = make_float2(__uint_as_float(raw.x), __uint_as_float(raw.y));
          f[2 * w + 1] = make_float2(__uint_as_float(raw.z), __uint_as_float(raw.w));
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) v[2 * j] = f[j].x, v[2 * j + 1] = f[j].y;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = 0.f;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int e = at + j * blockDim.x;
      v[j] = e < H ? to_f32<T>(p[e]) : 0.f;
    }
  }
}
// A vector in x's type or in float32.
template <typename T, bool VEC>
__device__ __forceinline__ void load8_as(const void* p, bool f32, int at, int H, float (&v)[8]) {
  if (f32) load8<float, VEC>(static_cast<const float*>(p), at, H, v);
  else load8<T, VEC>(static_cast<const T*>(p), at, H, v);
}

template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* p, int at, int H, const float (&v)[8]) {
  if constexpr (VEC) {
    if (at >= H) return;
    T e[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) e[j] = from_f32<T>(v[j]);
#pragma unroll
    for (int w = 0; w < (int)sizeof(T) / 2; ++w) reinterpret_cast<uint4*>(p + at)[w] = reinterpret_cast<uint4*>(e)[w];
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (at + j * (int)blockDim.x < H) p[at + j * blockDim.x] = from_f32<T>(v[j]);
  }
}

// Sum and maximum over the CTA, the same bits in every thread.  `red`: 64 floats that nobody has read since the last barrier.
__device__ __forceinline__ float2 block_sum_max(float s, float m, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) red[warp] = s, red[32 + warp] = m;
  __syncthreads();
  const bool live = lane < (blockDim.x >> 5);
  s = live ? red[lane] : 0.f;
  m = live ? red[32 + lane] : 0.f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  }
  return make_float2(s, m);
}

// (mean of squares + eps)^-1/2 of a row held in `v`, whose sum of squares is `ss`.  Where that exceeds float32 the squares of
// the row times 2^-80 are summed instead, which neither exceed nor fall below what float32 holds and beside which eps does not count
// (every thread of the CTA takes the same way: ss has the same bits everywhere).
template <int NV>
__device__ __forceinline__ float inverse_root(const float (&v)[NV][8], float ss, int H, float eps, float* red) {
  if (ss < 3e38f) return __frsqrt_rn(ss / (float)H + eps);
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) s = __fmaf_rn(v[i][j] * 0x1p-80f, v[i][j] * 0x1p-80f, s);
  __syncthreads();
  s = block_sum_max(s, 0.f, red).x;
  return 0x1p-80f * __frsqrt_rn(s / (float)H);
}

// round(127 t / top) of an element that lies next to a border between two codes, or whose factor 127 / top float32 does not
// hold.  The product by 127 is exact and the quotient of two float32 numbers is never nearer to a half-integer than 64 bits can
// tell, unless it is one.
__device__ __forceinline__ int code_exact(float t, float top) {
  const double q = 127.0 * (double)t / (double)top;
  return q == q ? max(-127, min(127, __double2int_rn(q))) : 0;
}

// One CTA per row, the row in registers (NV units of eight elements a thread), so that everything is read once, all loads of
// a thread in flight together:
//   p = x * (mean(x^2) + eps)^-1/2 * (post + offset)        (with `post`; x otherwise)
//   h = residual_scale * residual + scale * gate * p         rounded to the stream's type R, and stored
//   z = h * (mean(h^2) + eps)^-1/2 * (weight + offset)       of the rounded h
// in float32.  QUANT: INT8 rows instead of z.  The root is the same for a whole row, so it cancels out of
// codes = round(127 z / max|z|): with t = h * (weight + offset) they are round(127 t / max|t|), exactly (t is a float32
// product, exact where both factors have 16 bits), and the root goes into the row's scale alone, max|t| * root / 127: one reduction for
// the sum and the maximum, and codes that do not hang on the order of a sum.
// Bound by memory at many rows, by the chain of launch, load, reduction(s) and store at few.
template <typename T, typename R, int NV, bool VEC, bool QUANT>
__global__ void __launch_bounds__(512, 1)
block_norm_kernel(const NormArgs a) {
  __shared__ float red[3][64];
  allow_dependents();
  dependency_wait();
  const long m = blockIdx.x, outer = m / a.inner, inner = m - outer * a.inner;
  const int H = a.H;
  const T* x = static_cast<const T*>(a.x) + outer * a.xs.outer + inner * a.xs.inner;
  float v[NV][8], u[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i) load8<T, VEC>(x, unit_at<VEC>(i), H, v[i]);
  if (a.residual) {
    const R* r = static_cast<const R*>(a.residual) + outer * a.rs.outer + inner * a.rs.inner;
#pragma unroll
    for (int i = 0; i < NV; ++i) load8<R, VEC>(r, unit_at<VEC>(i), H, u[i]);
  }
  if (a.post) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) s = __fmaf_rn(v[i][j], v[i][j], s);
    s = block_sum_max(s, 0.f, red[0]).x;
    const float root = inverse_root(v, s, H, a.eps, red[0]);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float w[8];
      load8_as<T, VEC>(a.post, a.post_f32, unit_at<VEC>(i), H, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = v[i][j] * root * (w[j] + a.offset);
    }
  }
  if (a.gate) {
    const long at = outer * a.gs.outer + inner * a.gs.inner;
    if (a.gate_step) {
      const void* g = a.gate_f32 ? (const void*)(static_cast<const float*>(a.gate) + at) : static_cast<const T*>(a.gate) + at;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float w[8];
        load8_as<T, VEC>(g, a.gate_f32, unit_at<VEC>(i), H, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] *= w[j];
      }
    } else {
      const float g = a.gate_f32 ? static_cast<const float*>(a.gate)[at] : to_f32<T>(static_cast<const T*>(a.gate)[at]);
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] *= g;
    }
  }
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float h = v[i][j] * a.scale;
      if (a.residual) h = __fmaf_rn(a.residual_scale, u[i][j], h);
      h = to_f32<R>(from_f32<R>(h));
      const bool in = VEC || unit_at<VEC>(i) + j * (int)blockDim.x < H;   // (what is no element is 0: 0 * a gate that is none)
      v[i][j] = in ? h : 0.f;
      ss = __fmaf_rn(v[i][j], v[i][j], ss);
    }
  if (a.h) {
    R* h = static_cast<R*>(a.h) + m * H;
#pragma unroll
    for (int i = 0; i < NV; ++i) store8<R, VEC>(h, unit_at<VEC>(i), H, v[i]);
  }
  float top = 0.f;
  if constexpr (QUANT) {   // u: the rows times the weight
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float w[8];
      if (a.weight) load8_as<T, VEC>(a.weight, a.weight_f32, unit_at<VEC>(i), H, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        u[i][j] = a.weight ? v[i][j] * (w[j] + a.offset) : v[i][j];
        top = fmaxf(top, fabsf(u[i][j]));
      }
    }
  }
  const float2 both_of = block_sum_max(ss, top, red[1]);
  const float root = inverse_root(v, both_of.x, H, a.eps, red[2]);
  if constexpr (!QUANT) {
    T* z = static_cast<T*>(a.z) + m * H;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float w[8];
      if (a.weight) load8_as<T, VEC>(a.weight, a.weight_f32, unit_at<VEC>(i), H, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = a.weight ? v[i][j] * root * (w[j] + a.offset) : v[i][j] * root;
      store8<T, VEC>(z, unit_at<VEC>(i), H, w);
    }
  } else {
    top = both_of.y;
    if (threadIdx.x == 0) a.q_scale[m] = __fdiv_rn(top * root, 127.0f);
    const float inv = __fdiv_rn(127.0f, top);
    int8_t* q = a.q + m * H;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float2 t[4], r[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) t[j] = make_float2(u[i][2 * j], u[i][2 * j + 1]);
      const bool safe = inv < 3e38f && round_quotients(t, inv, r);
      uint32_t c[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) c[2 * j] = __float_as_uint(r[j].x), c[2 * j + 1] = __float_as_uint(r[j].y);
      if (!safe) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (!(inv < 3e38f) || !near_integer(u[i][j], inv)) c[j] = (uint32_t)code_exact(u[i][j], top);
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
          if (at + j * (int)blockDim.x < H) q[at + j * blockDim.x] = (int8_t)c[j];
      }
    }
  }
}

template <typename T, typename R, int NV>
static cudaError_t launch_norm(const NormArgs& a, int rows, int threads, bool vec, cudaStream_t st) {
  if (vec)
    return a.q ? launch_overlapped(block_norm_kernel<T, R, NV, true, true>, dim3(rows), dim3(threads), 0, st, a)
               : launch_overlapped(block_norm_kernel<T, R, NV, true, false>, dim3(rows), dim3(threads), 0, st, a);
  return a.q ? launch_overlapped(block_norm_kernel<T, R, NV, false, true>, dim3(rows), dim3(threads), 0, st, a)
             : launch_overlapped(block_norm_kernel<T, R, NV, false, false>, dim3(rows), dim3(threads), 0, st, a);
}

template <typename T, typename R>
static cudaError_t launch_norm_nv(const NormArgs& a, int rows, bool vec, cudaStream_t st) {
  int threads = 0;
  switch (row_units_per_thread(rows, (a.H + 7) / 8, 8, 256, 512, &threads)) {
    case 1: return launch_norm<T, R, 1>(a, rows, threads, vec, st);
    case 2: return launch_norm<T, R, 2>(a, rows, threads, vec, st);
    case 4: return launch_norm<T, R, 4>(a, rows, threads, vec, st);
    default: return launch_norm<T, R, 8>(a, rows, threads, vec, st);
  }
}

}  // namespace lq

extern "C" int lq_block_norm(const void* x, int x_dtype, long x_outer, long x_inner, const void* residual, int stream_dtype,
                             long r_outer, long r_inner, const void* gate, int gate_dtype, long g_outer, long g_inner,
                             int gate_step, const void* weight, int weight_dtype, const void* post, int post_dtype, void* z,
                             int8_t* q, float* q_scale, void* h, int rows, int inner, int H, float eps, float scale,
                             float residual_scale, float offset, void* stream) {
  using namespace lq;
  if (!x || rows <= 0 || inner <= 0 || H <= 0 || x_dtype < 0 || x_dtype > 2 || (z == nullptr) == (q == nullptr) ||
      (q != nullptr) != (q_scale != nullptr))
    return LQ_ERR_BAD_ARG;
  if (stream_dtype != x_dtype && !(residual && stream_dtype == LQ_DT_F32)) return LQ_ERR_BAD_ARG;
  const int side[3][2] = {{gate != nullptr, gate_dtype}, {weight != nullptr, weight_dtype}, {post != nullptr, post_dtype}};
  for (const auto& s : side)
    if (s[0] && s[1] != x_dtype && s[1] != LQ_DT_F32) return LQ_ERR_BAD_ARG;
  if (gate && gate_step != 0 && gate_step != 1) return LQ_ERR_BAD_ARG;
  if (!(eps >= 0.f)) return LQ_ERR_BAD_ARG;
  if (H > 32768) return LQ_ERR_SHAPE;
  NormArgs a = {};
  a.x = x, a.residual = residual, a.gate = gate, a.weight = weight, a.post = post;
  a.z = z, a.q = q, a.q_scale = q_scale, a.h = h;
  a.xs = {x_outer, x_inner}, a.rs = {r_outer, r_inner}, a.gs = {g_outer, g_inner};
  a.gate_step = gate_step, a.inner = inner, a.H = H;
  a.eps = eps, a.scale = scale, a.residual_scale = residual_scale, a.offset = offset;
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
  if (x_dtype == LQ_DT_F32) e = launch_norm_nv<float, float>(a, rows, vec, st);
  else if (x_dtype == LQ_DT_BF16)
    e = stream_dtype == LQ_DT_F32 ? launch_norm_nv<__nv_bfloat16, float>(a, rows, vec, st)
                                  : launch_norm_nv<__nv_bfloat16, __nv_bfloat16>(a, rows, vec, st);
  else
    e = stream_dtype == LQ_DT_F32 ? launch_norm_nv<__half, float>(a, rows, vec, st)
                                  : launch_norm_nv<__half, __half>(a, rows, vec, st);
  if (e != cudaSuccess) {
    record_cuda_error(e, "block_norm_kernel");
    return LQ_ERR_CUDA;
  }
  return check_launch("block_norm_kernel");
}
