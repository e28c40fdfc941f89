// kern_rope.cuh -- rotary positions as an operator of its own: both layouts
// of picolm's rope() (tensor.c:537-601), part of the head, scaled
// frequencies, FP32 / FP16 / BF16 rows, forward and adjoint.
//
//   y_a = x_a c - x_b s,  y_b = x_a s + x_b c,  c, s = gain * (cos, sin)(pos f_i)
//
// for the pairs (a, b) = (2i, 2i+1) (LLaMA) or (i, i + dim/2) (Qwen), i <
// dim/2; elements past dim pass through.  The adjoint (the gradient with
// respect to x) is the same with -s.  There is no table of positions: the
// angle is taken in FP64, so a position may be any non-negative int.
//
// Should be bound by HBM, as each element is read and written once; is bound by
// the start of its blocks.  A block rotates all
// heads of a few rows, so that the FP64 cosines (about a hundred instructions
// each) are computed once per (row, pair) into shared memory and not once
// per head.  8192 rows of 32 + 8 heads of 128 in BF16, half of each rotated
// (168 MB), on one B200: 46 us, 3.7 TB/s, 57% of a copy; the rest is a block's
// start, whose cosines and first rows nothing else of the block overlaps.
// On the way: an element a thread 125 us; runs of 16 bytes 78; a thread's
// place found once for all rows 53; blocks of equal width, two rows under
// way instead of four for more blocks an SM 46.  64 FP32 rows: 10 us.
#pragma once
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/pl_attn.h"

namespace pl {

constexpr int kRopeThreads = 256;  // at most
constexpr int kRopeRows = 8;  // rows per block, at most

// Cosine and sine of a pair at position pos, times the gain, rounded once
// from FP64 to FP32.
__device__ __forceinline__ float2 rope_cs(double half_turns, double gain, int pos) {
  double s, c;
  sincospi(half_turns * static_cast<double>(pos), &s, &c);
  return make_float2(static_cast<float>(c * gain), static_cast<float>(s * gain));
}

// The same in FP32 after an exact reduction to [-1, 1] half turns in FP64:
// within 2e-7 of rope_cs, at a tenth of its time.  For q, which no rounding
// to 8 bits follows.
__device__ __forceinline__ float2 rope_cs_fast(double half_turns, double gain, int pos) {
  const double x = half_turns * static_cast<double>(pos);
  float s, c;
  sincospif(static_cast<float>(x - 2.0 * rint(0.5 * x)), &s, &c);
  const float g = static_cast<float>(gain);
  return make_float2(c * g, s * g);
}

// Eight consecutive elements as FP32 (16-byte aligned FP16 / BF16, 32-byte
// spans of FP32).
__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
  x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
__device__ __forceinline__ void load8(const __half* p, float (&x)[8]) {
  const uint4 v = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    x[2 * i] = f.x, x[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&x)[8]) {
  const uint4 v = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void store8(__half* p, const float (&x)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&x)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

// Eight elements as they are in memory.
template <typename T>
struct Raw8 {
  uint4 v[sizeof(T) / 2];
};
template <typename T>
__device__ __forceinline__ Raw8<T> raw8(const T* p) {
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
    r.v[i] = reinterpret_cast<const uint4*>(p)[i];
  return r;
}
template <typename T>
__device__ __forceinline__ void unpack8(const Raw8<T>& r, float (&x)[8]) {
  load8(reinterpret_cast<const T*>(r.v), x);
}

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void from_f32(float* p, float x) { *p = x; }
__device__ __forceinline__ void from_f32(__half* p, float x) { *p = __float2half_rn(x); }
__device__ __forceinline__ void from_f32(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

struct RopeRowsArgs {
  pl_rope rope;
  const int* pos;
  int n, n_heads, n_kv_heads, adjoint, rows_per_block;
  int units, per_head;   // vector units of a row, of a head
  uint64_t per_head_inv; // ceil(2^32 / per_head)
  const void *q, *k;
  void *qo, *ko;
  long long q_stride, qo_stride, k_stride, ko_stride;  // elements between rows
};

// Place of pair i in a table of n (a multiple of 8) pairs.  Neighbouring lanes
// rotate neighbouring runs of eight elements, four pairs (LLaMA) or eight
// (Qwen) apart: what they read together lies side by side here, free of
// bank conflicts.
template <bool LLAMA>
__device__ __forceinline__ int pair_place(int i, int n) {
  return LLAMA ? (i & 3) * (n / 4) + (i >> 2) : (i & 7) * (n / 8) + (i >> 3);
}

// Cosines and sines of the block's rows, once for all heads.
template <bool LLAMA>
__device__ __forceinline__ void rope_rows_table(const RopeRowsArgs& a, int row0, int rows,
                                                float2 (*s_cs)[PL_ROPE_MAX_PAIRS],
                                                double* s_turns) {
  const int half = a.rope.dim >> 1;
  for (int i = threadIdx.x; i < half; i += blockDim.x) s_turns[i] = a.rope.half_turns[i];
  __syncthreads();
  for (int t = threadIdx.x; t < rows * half; t += blockDim.x) {
    const int r = t / half, i = t - r * half;
    float2 cs = rope_cs(s_turns[i], a.rope.gain, a.pos[row0 + r]);
    if (a.adjoint) cs.y = -cs.y;
    s_cs[r][pair_place<LLAMA>(i, PL_ROPE_MAX_PAIRS)] = cs;
  }
  __syncthreads();
}

// y = x rotated by cs, with the roundings of rope() (two products, a sum)
__device__ __forceinline__ void rope_one(float& a, float& b, float2 cs) {
  const float u = a, v = b;
  a = __fsub_rn(__fmul_rn(u, cs.x), __fmul_rn(v, cs.y));
  b = __fadd_rn(__fmul_rn(u, cs.y), __fmul_rn(v, cs.x));
}

// Any dim, stride and alignment: a unit is one pair, or one element past
// dim, of one head.
template <typename T>
__global__ void __launch_bounds__(kRopeThreads) rope_rows_any_kernel(
    const __grid_constant__ RopeRowsArgs a) {
  __shared__ float2 s_cs[kRopeRows][PL_ROPE_MAX_PAIRS];
  __shared__ double s_turns[PL_ROPE_MAX_PAIRS];
  const int hd = a.rope.head_dim, half = a.rope.dim >> 1;
  const int row0 = blockIdx.x * a.rows_per_block;
  const int rows = min(a.rows_per_block, a.n - row0);
  rope_rows_table<true>(a, row0, rows, s_cs, s_turns);
  const int heads = a.n_heads + a.n_kv_heads;
  const int per_head = half + (hd - a.rope.dim);
  for (int t = threadIdx.x; t < rows * heads * per_head; t += kRopeThreads) {
    const int u = t % per_head, rh = t / per_head, h = rh % heads, r = rh / heads;
    const bool is_q = h < a.n_heads;
    const long long row = row0 + r;
    const T* x = is_q ? static_cast<const T*>(a.q) + row * a.q_stride + h * hd
                      : static_cast<const T*>(a.k) + row * a.k_stride + (h - a.n_heads) * hd;
    T* y = is_q ? static_cast<T*>(a.qo) + row * a.qo_stride + h * hd
                : static_cast<T*>(a.ko) + row * a.ko_stride + (h - a.n_heads) * hd;
    if (u < half) {
      const bool llama = a.rope.type == PL_ROPE_LLAMA;
      const int ea = llama ? 2 * u : u, eb = llama ? 2 * u + 1 : u + half;
      float xa = to_f32(x[ea]), xb = to_f32(x[eb]);
      rope_one(xa, xb, s_cs[r][pair_place<true>(u, PL_ROPE_MAX_PAIRS)]);
      from_f32(y + ea, xa);
      from_f32(y + eb, xb);
    } else {
      y[a.rope.dim + u - half] = x[a.rope.dim + u - half];
    }
  }
}

// Aligned rows.  A unit is eight elements of a head (LLaMA; past dim: copied)
// or the two runs of eight that rotate together (Qwen, dim / 2 a multiple of
// eight).  A thread keeps its unit over the block's rows, so its place is
// found once, and has the loads of four (Qwen: two, of two runs) rows under
// way.
template <typename T, bool LLAMA>
__global__ void __launch_bounds__(kRopeThreads, sizeof(T) == 4 ? 2 : 3) rope_rows_kernel(
    const __grid_constant__ RopeRowsArgs a) {
  __shared__ float2 s_cs[kRopeRows][PL_ROPE_MAX_PAIRS];
  __shared__ double s_turns[PL_ROPE_MAX_PAIRS];
  const int hd = a.rope.head_dim, half = a.rope.dim >> 1;
  const int row0 = blockIdx.x * a.rows_per_block;
  const int rows = min(a.rows_per_block, a.n - row0);
  const int u = blockIdx.y * blockDim.x + threadIdx.x;
  const bool mine = u < a.units;
  const int h = static_cast<int>((static_cast<uint64_t>(u) * a.per_head_inv) >> 32);
  const int c = u - h * a.per_head;
  // Qwen: the runs below half, then those past dim
  const int el = LLAMA || c * 8 < half ? c * 8 : c * 8 + half;
  const bool two = !LLAMA && el < half, turns = el < a.rope.dim;
  const bool is_q = h < a.n_heads;
  const long long at = static_cast<long long>(is_q ? h : h - a.n_heads) * hd + el;
  const long long in_step = is_q ? a.q_stride : a.k_stride;
  const long long out_step = is_q ? a.qo_stride : a.ko_stride;
  const T* src = static_cast<const T*>(is_q ? a.q : a.k) + row0 * in_step + at;
  T* dst = static_cast<T*>(is_q ? a.qo : a.ko) + row0 * out_step + at;
  constexpr int U = LLAMA ? 4 : 2;
  Raw8<T> x[U], z[U];
  auto fetch = [&](int r0) {
#pragma unroll
    for (int k = 0; k < U; ++k)
      if (mine && r0 + k < rows) {
        x[k] = raw8(src + (r0 + k) * in_step);
        if (two) z[k] = raw8(src + (r0 + k) * in_step + half);
      }
  };
  fetch(0);  // on their way while the cosines are computed
  rope_rows_table<LLAMA>(a, row0, rows, s_cs, s_turns);
#pragma unroll 1
  for (int r0 = 0; r0 < rows; r0 += U) {
    if (r0) fetch(r0);
#pragma unroll
    for (int k = 0; k < U; ++k) {
      if (!mine || r0 + k >= rows) break;
      float y[8];
      unpack8(x[k], y);
      const float2* cs = s_cs[r0 + k];
      if constexpr (LLAMA) {
        if (turns) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (el + 2 * i < a.rope.dim)
              rope_one(y[2 * i], y[2 * i + 1],
                       cs[pair_place<true>((el >> 1) + i, PL_ROPE_MAX_PAIRS)]);
        }
      } else if (two) {
        float w[8];
        unpack8(z[k], w);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          rope_one(y[i], w[i], cs[pair_place<false>(el + i, PL_ROPE_MAX_PAIRS)]);
        store8(dst + (r0 + k) * out_step + half, w);
      }
      store8(dst + (r0 + k) * out_step, y);
    }
  }
}

}  // namespace pl
