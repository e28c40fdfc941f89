// kern_kv8_attn.cuh -- causal attention over the 8-bit paged cache.
//
// Entry i has n_tok query tokens, the last of them at row len - 1 of its
// slot; token j attends rows [0, len - n_tok + j] (none: its output is 0).
//
//   s_r = q . (code_r * sk_b) / sqrt(head_dim),  b = block of row r
//   o   = sum_r 2^(s_r log2e - m) sv_b code_r / sum_r 2^(s_r log2e - m)
#pragma once
#include <cstdint>

#include "kern_kv8.cuh"

namespace pl {

struct Kv8AttnArgs {
  Kv8Geo g;
  pl_rope rope;
  int n, total, max_tok, n_heads, group;
  const int *seqs, *start;
  const void* q;
  void* out;
  long long q_stride, out_stride;
  float score_scale;  // log2(e) / sqrt(head_dim)
};

constexpr int kKv8MaxGroup = 8;  // query heads per KV head

// One block per (token, KV head, entry): the plain form, a page at a time.
constexpr int kPlainThreads = 128;

template <typename T, int HD, int FMT>
__global__ void __launch_bounds__(kPlainThreads) kv8_attend_plain_kernel(
    const __grid_constant__ Kv8AttnArgs a) {
  __shared__ float s_q[kKv8MaxGroup][HD];
  __shared__ float s_p[kKv8MaxGroup][kPage];
  __shared__ float s_alpha[kKv8MaxGroup], s_m[kKv8MaxGroup], s_l[kKv8MaxGroup];
  __shared__ float2 s_cs[HD / 2];
  const int tid = threadIdx.x, h = blockIdx.y, G = a.group;
  Kv8Entry e;
  if (!kv8_entry(a.g, blockIdx.z, a.total, a.max_tok, a.seqs, a.start, e)) {
    if (tid == 0 && blockIdx.x == 0 && h == 0) atomicOr(&a.g.head->err, ERR_BAD_ARG);
    return;
  }
  const int j = blockIdx.x;
  if (j >= e.n_tok) return;
  const int pos = e.len - e.n_tok + j;
  const T* q = static_cast<const T*>(a.q) + (e.tok0 + j) * a.q_stride + h * G * HD;
  T* out = static_cast<T*>(a.out) + (e.tok0 + j) * a.out_stride + h * G * HD;
  if (pos < 0) {
    for (int t = tid; t < G * HD; t += kPlainThreads) from_f32(out + t, 0.f);
    return;
  }
  for (int i = tid; i < a.rope.dim >> 1; i += kPlainThreads) s_cs[i] = rope_cs_fast(a.rope, i, pos);
  __syncthreads();
  for (int t = tid; t < G * (HD / 8); t += kPlainThreads) {
    const int gq = t / (HD / 8), el = (t % (HD / 8)) * 8;
    float x[8];
    load_rotated<T, HD>(q + gq * HD, el, a.rope, s_cs, x);
    for (int i = 0; i < 8; ++i) s_q[gq][el + i] = x[i] * a.score_scale;
  }
  if (tid < G) s_m[tid] = -INFINITY, s_l[tid] = 0.f;
  float o[kKv8MaxGroup] = {};
  __syncthreads();
  for (int r0 = 0; r0 <= pos; r0 += kPage) {
    const int page = a.g.table[static_cast<long long>(e.slot) * a.g.max_pages + r0 / kPage];
    if (page < 0 || page >= a.g.n_pages) {
      if (tid == 0) atomicOr(&a.g.head->err, ERR_BAD_ARG);
      return;
    }
    const long long ks = a.g.slab(page, h, 0);
    const int rows = min(kPage, pos + 1 - r0);
    for (int t = tid; t < G * kPage; t += kPlainThreads) {
      const int r = t % kPage, gq = t / kPage;
      float s = -INFINITY;
      if (r < rows) {
        s = 0.f;
        const uint8_t* kr = a.g.codes + (ks * kPage + r) * HD;
        for (int el = 0; el < HD; el += 8) {
          float x[8];
          decode8<FMT>(*reinterpret_cast<const uint2*>(kr + el), x);
          for (int i = 0; i < 8; ++i) s += s_q[gq][el + i] * x[i];
        }
        s *= a.g.scales[ks * kBlocksPerPage + r / kBlock];
      }
      s_p[gq][r] = s;
    }
    __syncthreads();
    for (int gq = tid >> 5; gq < G; gq += kPlainThreads / 32) {
      const int lane = tid & 31;
      const float s0 = s_p[gq][lane], s1 = s_p[gq][lane + 32];
      float m = fmaxf(s0, s1);
      for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
      m = fmaxf(m, s_m[gq]);
      const float p0 = exp2f(s0 - m), p1 = exp2f(s1 - m);
      float l = p0 + p1;
      for (int d = 16; d > 0; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
      s_p[gq][lane] = p0 * a.g.scales[(ks + 1) * kBlocksPerPage + lane / kBlock];
      s_p[gq][lane + 32] = p1 * a.g.scales[(ks + 1) * kBlocksPerPage + (lane + 32) / kBlock];
      __syncwarp();
      if (lane == 0) {
        s_alpha[gq] = exp2f(s_m[gq] - m);
        s_l[gq] = s_l[gq] * s_alpha[gq] + l;
        s_m[gq] = m;
      }
    }
    __syncthreads();
    if (tid < HD) {
      for (int gq = 0; gq < G; ++gq) o[gq] *= s_alpha[gq];
      for (int r = 0; r < rows; ++r) {
        uint2 c = make_uint2(a.g.codes[((ks + 1) * kPage + r) * HD + tid], 0u);
        float x[8];
        decode8<FMT>(c, x);
        for (int gq = 0; gq < G; ++gq) o[gq] += s_p[gq][r] * x[0];
      }
    }
    __syncthreads();
  }
  if (tid < HD)
    for (int gq = 0; gq < G; ++gq) from_f32(out + gq * HD + tid, o[gq] / s_l[gq]);
}

}  // namespace pl
