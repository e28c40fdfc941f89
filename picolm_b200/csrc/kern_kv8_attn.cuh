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

// ------------------------------------------------------- one token a slot
// Bound by HBM: 2 * head_dim + 0.5 bytes a row and KV head.
//
// Work partition.  A tile is kTileRows rows of one page and KV head, 4 KB of
// K and 4 KB of V.  The tiles of all entries, (entry, head, tile) in order,
// form one list; every block takes an equal contiguous slice of it and every
// warp of the block one of that, whatever the lengths are.  The part of one
// (entry, head) -- a run -- inside a warp's slice is a segment.
//
// Each warp is on its own: its first lane streams the warp's tiles through a
// ring of kStages 8 KB stages (tiled TMA loads, swizzled by the width of a
// row so that ldmatrix is free of bank conflicts), and the whole warp
// consumes them, so no warp waits for another until its slice is done.
//
// Scores and P.V run on mma.sync (m16n8k16, FP16 in, FP32 out): on CUDA
// cores the dot products alone would need more issue slots than HBM leaves.
// Every code is exact in FP16.  ldmatrix moves the bytes as 16-bit pairs:
// without .trans a thread gets bytes 4c .. 4c+3 of a row's 16-byte chunk, so
// K step j of Q K^T holds the dims 16j + 4c + {0, 1, 2, 3} in its slots 2c,
// 2c+1, 2c+8, 2c+9 (q is laid out the same way); with .trans it gets bytes 2g, 2g+1
// of rows 2c, 2c+1, so two n-tiles of P V hold the even and the odd dims of
// a chunk.  Rows 0..7 of the A operand hold the FP16 high part of q (of the
// weights), rows 8..15 the residual, which costs nothing in an m16 tile of
// at most 8 heads and carries FP32 inputs to 2^-22.
//
// Ranges.  q is scaled by the power of two that puts its row's largest
// element into [1, 2); weights are 2^(s - m) * sv * 2^14 / ref with ref the
// largest V scale so far, so that residuals stay above FP16's smallest
// subnormals (a weight of 2^-20 still has 18 bits) and nothing overflows.
// Each tile's P V starts from zero and is added to the running output with
// one rounded FP32 FMA: the tensor core truncates as it accumulates, and
// over a long segment that would add up in one direction.
//
// On one B200: 64 sequences of 2048 rows, 32/4 heads of 64, FP32: 26 us (69
// MB); 32 ragged ones up to 8192 rows, 32/8 heads of 128, BF16: 85 us (335
// MB, 3.9 TB/s); one of 32768, 32/8 of 64: 19 us; one of 256 rows: 10 us.
// Streaming takes 11 of the 26 us at a copy's rate; before it a block reads
// and scans the books, finds its first tile and rotates q, and after it the
// runs that cross blocks are merged.  At head_dim 128
// the stream runs at the pace of its eight warps, which have 255 registers
// each; more warps spill and are slower, as were four of 64-row tiles.
//
// Segments of a run in several warps of a block are merged in shared
// memory by the warp where the run starts; runs over several blocks leave
// one partial a block in the workspace, and the block that finishes a run's
// last partial merges them, in the order of the blocks.
constexpr float kWeightScale = 16384.f;
constexpr float kMinRef = 1e-30f;

template <int W, int TR, int NS, int HD>
struct DecShapeT {
  static constexpr int kWarps = W;
  static constexpr int kThreads = W * 32;
  static constexpr int kTileRows = TR;
  static constexpr int kTileBytes = TR * HD;              // of K, and of V
  static constexpr int kTilesPerPage = kPage / kTileRows;
  static constexpr int kBlocks = kTileRows / kBlock;      // scales in a tile
  static constexpr int kStages = NS;
  static constexpr int kPartFloats = 32 * (HD / 4) + 16;  // a partial: o lane-wise, then m, l
};

template <int HD>
struct DecShape : DecShapeT<8, 64, 3, 64> {};
template <>
struct DecShape<128> : DecShapeT<8, 32, 2, 128> {};

template <int HD>
struct DecSmem {
  using Sh = DecShape<HD>;
  uint8_t ring[Sh::kWarps][Sh::kStages][2][Sh::kTileBytes];  // 1024-byte aligned
  float scales[Sh::kWarps][Sh::kStages][2][kBlocksPerPage];
  float part[Sh::kWarps][Sh::kPartFloats];
  float2 cs[Sh::kWarps][HD / 2];
  double half_turns[HD / 2];
  uint64_t full[Sh::kWarps][Sh::kStages];
  int prefix[kPlanSeqs + 1], slot[kPlanSeqs], len[kPlanSeqs];
  int warp_sum[Sh::kWarps];
  int ended[4];   // of the run that an earlier block began: run, first, last tile, warp that has it
  int finish[2];
};

struct Kv8DecodeArgs {
  Kv8AttnArgs a;
  const void *k, *v;  // one row an entry, appended first (APPEND)
  long long k_stride, v_stride;
  float* part;    // [2 * blocks][kPartFloats]
  int* arrived;   // [blocks], zero at rest: by the block where a run starts
};

// Four consecutive elements (16-byte aligned FP32, 8-byte aligned 16-bit).
__device__ __forceinline__ void load4(const float* p, float (&x)[4]) {
  const float4 v = *reinterpret_cast<const float4*>(p);
  x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
}
__device__ __forceinline__ void load4(const __half* p, float (&x)[4]) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  const float2 a = unpack_half2(v.x), b = unpack_half2(v.y);
  x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
}
__device__ __forceinline__ void load4(const __nv_bfloat16* p, float (&x)[4]) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  x[0] = __uint_as_float(v.x << 16), x[1] = __uint_as_float(v.x & 0xffff0000u);
  x[2] = __uint_as_float(v.y << 16), x[3] = __uint_as_float(v.y & 0xffff0000u);
}
__device__ __forceinline__ void store4(float* p, const float (&x)[4]) {
  *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
}
__device__ __forceinline__ void store4(__half* p, const float (&x)[4]) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_half2(x[0], x[1]), pack_half2(x[2], x[3]));
}
__device__ __forceinline__ void store4(__nv_bfloat16* p, const float (&x)[4]) {
  const __nv_bfloat162 a = __floats2bfloat162_rn(x[0], x[1]), b = __floats2bfloat162_rn(x[2], x[3]);
  *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a),
                                            *reinterpret_cast<const uint32_t*>(&b));
}

// A row's elements 16j + 4c .. + 3, and those they rotate with: all loads
// of a row are issued before one is used.
template <typename T, int HD>
struct QRow {
  float y[HD / 16][4], z[HD / 16][4];
  __device__ __forceinline__ void load(const T* x, int c, const pl_rope& r) {
    const int half = r.dim >> 1;
#pragma unroll
    for (int j = 0; j < HD / 16; ++j) load4(x + 16 * j + 4 * c, y[j]);
    if (r.type == PL_ROPE_QWEN) {
#pragma unroll
      for (int j = 0; j < HD / 16; ++j) {
        const int e = 16 * j + 4 * c;
        if (half % 4 == 0) {
          const int o = e < half ? e + half : e < r.dim ? e - half : e;
          load4(x + o, z[j]);
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int d = e + k;
            z[j][k] = to_f32(x[d < half ? d + half : d < r.dim ? d - half : d]);
          }
        }
      }
    }
  }
  // cs: cosine and sine of the pairs
  __device__ __forceinline__ void rotate(int c, const pl_rope& r, const float2* cs) {
    const int half = r.dim >> 1;
#pragma unroll
    for (int j = 0; j < HD / 16; ++j) {
      const int e = 16 * j + 4 * c;
      if (r.type == PL_ROPE_LLAMA) {
#pragma unroll
        for (int k = 0; k < 4; k += 2)
          if (e + k < r.dim) {
            const float2 f = cs[(e + k) >> 1];
            const float a = y[j][k], b = y[j][k + 1];
            y[j][k] = a * f.x - b * f.y;
            y[j][k + 1] = a * f.y + b * f.x;
          }
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int d = e + k;
          if (d < r.dim) {
            const float2 f = cs[d < half ? d : d - half];
            y[j][k] = d < half ? y[j][k] * f.x - z[j][k] * f.y : z[j][k] * f.y + y[j][k] * f.x;
          }
        }
      }
    }
  }
};

// Codes as FP16 pairs.  int8: the byte with its sign bit flipped below a
// 0x64 is 1024 + 128 + code in FP16; e4m3 converts in hardware.
template <int FMT, int SEL>
__device__ __forceinline__ uint32_t codes_half2(uint32_t w) {
  // bytes a, b of w with SEL = a | b << 4
  if constexpr (FMT == PL_KV8_INT8) {
    constexpr uint32_t sel = (SEL & 0xf) | 0x40 | ((SEL >> 4) << 8) | 0x4000;
    const uint32_t h = __byte_perm(w ^ 0x80808080u, 0x64646464u, sel);
    uint32_t d;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(h), "r"(0x64806480u));
    return d;
  } else {
    constexpr uint32_t sel = (SEL & 0xf) | (SEL & 0xf0);
    uint32_t d;
    const uint16_t two = static_cast<uint16_t>(sel == 0x10 ? w : __byte_perm(w, 0u, sel | 0x4400u));
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(d) : "h"(two));
    return d;
  }
}

// Byte offset of 16-byte chunk `ch` of row r in a tile of HD-byte rows, as
// the TMA swizzle of that width places it.
template <int HD>
__device__ __forceinline__ uint32_t tile_off(int r, int ch) {
  if constexpr (HD == 64) return r * 64 + ((ch ^ ((r >> 1) & 3)) << 4);
  return r * 128 + ((ch ^ (r & 7)) << 4);
}

// Counts one arrival at a counter in global memory: what the warp (or block)
// wrote before, ordered by its own barrier, is visible to who counts later,
// and what earlier arrivals wrote to this thread.
__device__ __forceinline__ int arrive_acq_rel(int* counter) {
  int old;
  asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;"
               : "=r"(old)
               : "l"(counter)
               : "memory");
  return old;
}

// The list of tiles: prefix sums over entries, in tiles of all heads.
template <int HD>
struct DecWork {
  const int* prefix;
  int n, heads;
  int total, blocks;  // tiles; blocks that hold work
  __device__ __forceinline__ int begin(int b) const {
    return static_cast<int>(static_cast<long long>(b) * total / blocks);
  }
  // the block that owns tile x: the largest b with begin(b) <= x
  __device__ __forceinline__ int block_of(int x) const {
    return static_cast<int>(((static_cast<long long>(x) + 1) * blocks - 1) / total);
  }
  __device__ __forceinline__ int entry_of(int x) const {
    // right at once where the entries are alike
    int lo = static_cast<int>(static_cast<float>(x) * (static_cast<float>(n) /
                                                       static_cast<float>(total)));
    lo = min(lo, n - 1);
    if (prefix[lo] <= x && x < prefix[lo + 1]) return lo;
    lo = 0;
    int hi = n - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (prefix[mid + 1] > x) hi = mid; else lo = mid + 1;
    }
    return lo;
  }
};

// Running state of a segment: row g = lane / 4 of the A operand is query
// head g of the KV head; of each 16-byte chunk ch this thread holds the dims
// 16ch + 4(lane % 4) + {0, 2, 1, 3}, in o[4ch ..] (even and odd n-tile).
template <int HD>
struct DecState {
  float m, l, o[HD / 4];
  __device__ __forceinline__ void clear() {
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int i = 0; i < HD / 4; ++i) o[i] = 0.f;
  }
  __device__ __forceinline__ void fold(float m2, float l2, const float (&o2)[HD / 4]) {
    const float mx = fmaxf(m, m2);
    if (mx == -INFINITY) {  // neither has a row (or one holds NaN)
      l += l2;
      return;
    }
    const float a = ex2(m - mx), b = ex2(m2 - mx);
    l = l * a + l2 * b;
#pragma unroll
    for (int i = 0; i < HD / 4; ++i) o[i] = o[i] * a + o2[i] * b;
    m = mx;
  }
  __device__ __forceinline__ void save(float* p, int lane) const {
#pragma unroll
    for (int i = 0; i < HD / 4; ++i) p[i * 32 + lane] = o[i];
    if ((lane & 3) == 0) {
      p[8 * HD + (lane >> 2)] = m;
      p[8 * HD + 8 + (lane >> 2)] = l;
    }
  }
  __device__ __forceinline__ void fold_from(const float* p, int lane) {
    float o2[HD / 4];
    const float m2 = p[8 * HD + (lane >> 2)], l2 = p[8 * HD + 8 + (lane >> 2)];
#pragma unroll
    for (int i = 0; i < HD / 4; ++i) o2[i] = p[i * 32 + lane];
    fold(m2, l2, o2);
  }
  // Two partials from global memory (the second if `two`), loaded at once.
  __device__ __forceinline__ void fold_two(const float* p, const float* q, bool two, int lane) {
    float po[HD / 4], qo[HD / 4];
    const float pm = __ldcg(p + 8 * HD + (lane >> 2)), pl_ = __ldcg(p + 8 * HD + 8 + (lane >> 2));
    const float qm = __ldcg(q + 8 * HD + (lane >> 2)), ql = __ldcg(q + 8 * HD + 8 + (lane >> 2));
#pragma unroll
    for (int i = 0; i < HD / 4; ++i) {
      po[i] = __ldcg(p + i * 32 + lane);
      qo[i] = __ldcg(q + i * 32 + lane);
    }
    fold(pm, pl_, po);
    if (two) fold(qm, ql, qo);
  }
  template <typename T>
  __device__ __forceinline__ void write(T* out, int lane, int group) const {
    const int g = lane >> 2, c = lane & 3;
    if (g >= group) return;
    const float inv = 1.0f / l;
#pragma unroll
    for (int ch = 0; ch < HD / 16; ++ch) {
      const float x[4] = {o[4 * ch] * inv, o[4 * ch + 2] * inv, o[4 * ch + 1] * inv,
                          o[4 * ch + 3] * inv};
      store4(out + g * HD + 16 * ch + 4 * c, x);
    }
  }
};

// ---- a warp appends a row to a tile it holds
template <int FMT>
__device__ __forceinline__ uint32_t encode1(float x) {
  if constexpr (FMT == PL_KV8_INT8)
    return static_cast<uint32_t>(__float2int_rn(fminf(fmaxf(x, -127.f), 127.f))) & 0xffu;
  return __nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
}

// The quantisation of kv8_append_kernel for one new row `r` (of k or v) of a
// tile in shared memory, there and in global memory.  x: this lane's HD / 32
// consecutive elements, rotated; tile, gtile: the tile's row 0; block: first
// row of r's block; s_scale, g_scale: the block's scale.
template <int HD, int FMT>
__device__ __forceinline__ void append_row(const float (&x)[HD / 32], int lane, int r, int block,
                                           uint32_t tile, uint8_t* gtile, float* s_scale,
                                           float* g_scale) {
  constexpr int E = HD / 32;
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < E; ++j) top = max(top, __float_as_uint(fabsf(x[j])));
  top = __reduce_max_sync(0xffffffffu, top);
  const uint32_t old_bits = r > block ? __float_as_uint(*s_scale) : 0u;
  float s = __fdiv_rn(__uint_as_float(top), code_top<FMT>());
  if (top >= 0x7f800000u) s = __uint_as_float(0x7fc00000u);
  s = __uint_as_float(max(__float_as_uint(s), old_bits));
  const float by = s > 0.f ? s : 1.f;
  __syncwarp();  // every lane has read the old scale
  if (lane == 0) {
    *s_scale = s;
    *g_scale = s;
  }
  uint32_t code = 0;
#pragma unroll
  for (int j = 0; j < E; ++j)  // (+ 0: as quotient() has it, -0 becomes 0)
    code |= encode1<FMT>(__fdiv_rn(x[j], by) + 0.f) << (8 * j);
  if (!(s < INFINITY)) code = 0;  // no code stands for a NaN
  const int el = lane * E;
  const uint32_t at = tile + tile_off<HD>(r, el >> 4) + (el & 15);
  if constexpr (E == 2) {
    asm volatile("st.shared.u16 [%0], %1;" ::"r"(at), "h"(static_cast<uint16_t>(code)) : "memory");
    *reinterpret_cast<uint16_t*>(gtile + r * HD + el) = static_cast<uint16_t>(code);
  } else {
    asm volatile("st.shared.u32 [%0], %1;" ::"r"(at), "r"(code) : "memory");
    *reinterpret_cast<uint32_t*>(gtile + r * HD + el) = code;
  }
  if (__float_as_uint(s) != old_bits && r > block) {  // the scale has grown
    const float ratio = s > 0.f ? __fdiv_rn(__uint_as_float(old_bits), s) : 1.f;
    for (int o = lane * 8; o < (r - block) * HD; o += 256) {
      const int row = block + o / HD, e = o % HD;
      const uint32_t p = tile + tile_off<HD>(row, e >> 4) + (e & 15);
      uint2 c;
      asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(c.x), "=r"(c.y) : "r"(p) : "memory");
      float y[8];
      decode8<FMT>(c, y);
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = __fmul_rn(y[j], ratio);
      c = encode8<FMT>(y);
      asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(p), "r"(c.x), "r"(c.y) : "memory");
      *reinterpret_cast<uint2*>(gtile + row * HD + e) = c;
    }
  }
  __syncwarp();
}

template <typename T, int HD, int FMT, bool APPEND>
__global__ void __launch_bounds__(DecShape<HD>::kThreads, 1) kv8_decode_kernel(
    const __grid_constant__ Kv8DecodeArgs da, const __grid_constant__ CUtensorMap tm) {
  using Sh = DecShape<HD>;
  constexpr int W = Sh::kWarps, NS = Sh::kStages, TR = Sh::kTileRows;
  extern __shared__ uint8_t smem_raw[];
  DecSmem<HD>& sm = *reinterpret_cast<DecSmem<HD>*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const Kv8AttnArgs& a = da.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, c = lane & 3;
  const int heads = a.g.n_kv_heads, G = a.group;
  // the frequencies to shared memory: lanes of a warp want different ones
  if (tid < HD / 2) sm.half_turns[tid] = a.rope.half_turns[tid];
  if (lane == 0) {
    for (int s = 0; s < NS; ++s) mbar_init(&sm.full[warp][s], 1);
    fence_mbar_init();
    if (warp == 0) tma_prefetch_desc(&tm);
  }
  __syncwarp();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // ---- tiles of every entry, scanned
  {
    const int per = (a.n + Sh::kThreads - 1) / Sh::kThreads, i0 = tid * per;
    int mine = 0;
    bool bad = false;
    for (int i = i0; i < min(a.n, i0 + per); ++i) {
      Kv8Entry e;
      bool ok = kv8_entry(a.g, i, a.total, 1, a.seqs, a.start, e);
      if (APPEND) ok = ok && e.len > 0;
      bad |= !ok;
      const int rows = ok && e.n_tok ? e.len : 0;
      const int tiles = (rows + TR - 1) / TR * heads;
      sm.prefix[i] = tiles;
      sm.slot[i] = e.slot;
      sm.len[i] = rows;
      mine += tiles;
      // nothing to attend: zeros
      if (ok && e.n_tok && e.len == 0 && blockIdx.x == 0)
        for (int d = 0; d < a.n_heads * HD; ++d)
          from_f32(static_cast<T*>(a.out) + e.tok0 * a.out_stride + d, 0.f);
    }
    if (bad && blockIdx.x == 0) atomicOr(&a.g.head->err, ERR_BAD_ARG);
    int x = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, d);
      if (lane >= d) x += y;
    }
    if (lane == 31) sm.warp_sum[warp] = x;
    __syncthreads();
    int base = 0, total = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      base += w < warp ? sm.warp_sum[w] : 0;
      total += sm.warp_sum[w];
    }
    int run = base + x - mine;
    for (int i = i0; i < min(a.n, i0 + per); ++i) {
      const int t = sm.prefix[i];
      sm.prefix[i] = run;
      run += t;
    }
    if (tid == 0) {
      sm.prefix[a.n] = total;
      sm.finish[0] = sm.finish[1] = -1;
      sm.ended[0] = -1;
    }
    __syncthreads();
  }
  const int total = sm.prefix[a.n];
  // about a tile for each warp (9 tiles make two blocks of 4 and 5): fewer
  // blocks share a run then
  const DecWork<HD> work{sm.prefix, a.n, heads, total,
                         min(static_cast<int>(gridDim.x), (total + W - 1) / W)};
  const int blk = blockIdx.x;
  if (blk >= work.blocks) return;
  const int b0 = work.begin(blk), b1 = work.begin(blk + 1), span = b1 - b0;
  const int x0 = b0 + warp * span / W, x1 = b0 + (warp + 1) * span / W;

  // ---- this warp's tiles: 32 at a time, tile t_base + lane in this lane
  int t_run = 0, t_row = 0, t_slab = 0, t_base = x0;
  auto find_tile = [&](int base) -> int {  // the page, not yet checked
    t_base = base;
    const int x = base + lane;
    if (x >= x1) return 0;
    const int i = work.entry_of(x);
    const int tiles = (sm.prefix[i + 1] - sm.prefix[i]) / heads;
    const int rem = x - sm.prefix[i], h = rem / tiles, t = rem - h * tiles;
    t_run = i * heads + h;
    t_row = t * TR;
    return a.g.table[static_cast<long long>(sm.slot[i]) * a.g.max_pages + t / Sh::kTilesPerPage];
  };
  auto place_tile = [&](int page) {
    if (page < 0 || page >= a.g.n_pages) {
      atomicOr(&a.g.head->err, ERR_BAD_ARG);
      page = 0;  // read instead; a row is not appended there
    }
    t_slab = static_cast<int>(a.g.slab(page, t_run % heads, 0));
  };
  auto issue = [&](int x) {
    const int slab = __shfl_sync(0xffffffffu, t_slab, x - t_base);
    const int row = __shfl_sync(0xffffffffu, t_row, x - t_base);
    if (lane == 0) {
      const int s = (x - x0) % NS;
      uint64_t* bar = &sm.full[warp][s];
      mbar_arrive_expect_tx(bar, 2 * Sh::kTileBytes + 2 * kBlocksPerPage * 4);
      tma_load_3d(sm.ring[warp][s][0], &tm, bar, 0, row % kPage, slab);  // K and V
      bulk_load(sm.scales[warp][s], a.g.scales + static_cast<long long>(slab) * kBlocksPerPage,
                2 * kBlocksPerPage * 4, bar);
    }
  };
  // the query rows of a run, as they are in memory
  QRow<T, HD> q;
  auto load_q = [&](int run) {
    const int i = run / heads, h = run - i * heads, tok = a.start ? a.start[i] : i;
    q.load(static_cast<const T*>(a.q) + tok * a.q_stride + (h * G + min(g, G - 1)) * HD, c, a.rope);
  };
  bool ok = true;
  int issued = x0;
  if (x0 < x1) {
    const int page = find_tile(x0);
    load_q(__shfl_sync(0xffffffffu, t_run, 0));
    place_tile(page);
    for (; issued < x1 && issued < x0 + NS; ++issued) issue(issued);
  }

  uint32_t qa[HD / 16][4];
  DecState<HD> st;
  st.clear();
  float ref = kMinRef, q_scale = 0.f;
  int run = -1, run_first = 0, run_last = 0, len = 0;  // the current run and its tiles
  const uint32_t ring = smem_u32(sm.ring[warp]);
  // tiles are consumed a few behind the issued ones: a batch of their own
  int c_run = t_run, c_row = t_row, c_slab = t_slab, c_base = t_base;
  for (int x = x0; x < x1 && ok; ++x) {
    if (x - c_base >= 32) {
      c_run = t_run, c_row = t_row, c_slab = t_slab, c_base = t_base;
    }
    const int x_run = __shfl_sync(0xffffffffu, c_run, x - c_base);
    const int row0 = __shfl_sync(0xffffffffu, c_row, x - c_base);
    const int i = x_run / heads, h = x_run - i * heads;
    if (x_run != run) {
      // ---- a new run: its query rows, rotated, scaled and split
      run = x_run;
      const int tiles = (sm.prefix[i + 1] - sm.prefix[i]) / heads;
      run_first = sm.prefix[i] + h * tiles;
      run_last = run_first + tiles - 1;
      len = sm.len[i];
      if (x != x0) load_q(run);
      for (int p = lane; p < a.rope.dim >> 1; p += 32)
        sm.cs[warp][p] = rope_cs_fast(sm.half_turns[p], a.rope.gain, len - 1);
      __syncwarp();
      q.rotate(c, a.rope, sm.cs[warp]);
      __syncwarp();
      float top = 0.f;
#pragma unroll
      for (int j = 0; j < HD / 16; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(q.y[j][e]));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // 2^-e with 2^e <= top < 2^(e+1), for normal finite tops
      const uint32_t ex = __float_as_uint(top) >> 23;
      const bool norm = ex > 1 && ex < 253;
      const float down = g >= G ? 0.f : norm ? __uint_as_float((254u - ex) << 23) : 1.f;
      q_scale = (norm ? __uint_as_float(ex << 23) : 1.f) * a.score_scale;
#pragma unroll
      for (int j = 0; j < HD / 16; ++j)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf)
          split_hi_lo(q.y[j][2 * hf] * down, q.y[j][2 * hf + 1] * down, qa[j][2 * hf],
                      qa[j][2 * hf + 1]);
      st.clear();
      ref = kMinRef;
    }
    const int s = (x - x0) % NS;
    const uint32_t kt = ring + s * 2 * Sh::kTileBytes, vt = kt + Sh::kTileBytes;
    float* sk = sm.scales[warp][s][0] + row0 % kPage / kBlock;
    float* sv = sm.scales[warp][s][1] + row0 % kPage / kBlock;
    const int seen = len - row0;  // rows of the tile, at least 1
    // ---- the entry's new row belongs to this tile: fetched before the wait
    constexpr int E = HD / 32;
    float kx[E], vx[E];
    const bool appends = APPEND && seen <= TR;
    int page = -1;
    if (appends) {
      page = a.g.table[static_cast<long long>(sm.slot[i]) * a.g.max_pages + row0 / kPage];
      for (int p = lane; p < a.rope.dim >> 1; p += 32)
        sm.cs[warp][p] = rope_cs(sm.half_turns[p], a.rope.gain, len - 1);
      const T* k = static_cast<const T*>(da.k) + i * da.k_stride + h * HD;
      const T* v = static_cast<const T*>(da.v) + i * da.v_stride + h * HD;
      const int half = a.rope.dim >> 1;
      __syncwarp();
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const int d = lane * E + j;
        const float own = to_f32(k[d]);
        vx[j] = to_f32(v[d]);
        kx[j] = own;
        if (d < a.rope.dim) {
          const bool llama = a.rope.type == PL_ROPE_LLAMA;
          const bool first = llama ? !(d & 1) : d < half;
          const float other = to_f32(k[llama ? d ^ 1 : first ? d + half : d - half]);
          const float2 f = sm.cs[warp][llama ? d >> 1 : first ? d : d - half];
          kx[j] = first ? __fsub_rn(__fmul_rn(own, f.x), __fmul_rn(other, f.y))
                        : __fadd_rn(__fmul_rn(other, f.y), __fmul_rn(own, f.x));
        }
      }
    }
    if (!mbar_wait_warp(&sm.full[warp][s], ((x - x0) / NS) & 1)) {
      if (lane == 0) atomicOr(&a.g.head->err, ERR_TIMEOUT_FULL);
      ok = false;
      break;
    }
    if (appends && page >= 0 && page < a.g.n_pages) {
      const int r = seen - 1, block = r / kBlock * kBlock;
      const long long slab = __shfl_sync(0xffffffffu, c_slab, x - c_base);
      const int b = (row0 % kPage + block) / kBlock;
      uint8_t* gt = a.g.codes + (slab * kPage + row0 % kPage) * HD;
      append_row<HD, FMT>(kx, lane, r, block, kt, gt, &sm.scales[warp][s][0][b],
                          a.g.scales + slab * kBlocksPerPage + b);
      append_row<HD, FMT>(vx, lane, r, block, vt, gt + kPage * HD, &sm.scales[warp][s][1][b],
                          a.g.scales + (slab + 1) * kBlocksPerPage + b);
    }
    // ---- S = Q K^T
    float2 sc[TR / 8];  // this thread's columns 8nt + 2c, + 1 of row g
    float mt = -INFINITY;
#pragma unroll
    for (int nt = 0; nt < TR / 8; ++nt) {
      float acc[4];
#pragma unroll
      for (int q4 = 0; q4 < HD / 64; ++q4) {
        uint32_t w[4];
        ldmatrix_x4(kt + tile_off<HD>(nt * 8 + (lane & 7), 4 * q4 + (lane >> 3)), w[0], w[1], w[2],
                    w[3]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t b0 = codes_half2<FMT, 0x10>(w[j]), b1 = codes_half2<FMT, 0x32>(w[j]);
          if (q4 == 0 && j == 0) mma_16816_zero(acc, qa[0], b0, b1);
          else mma_16816(acc, qa[4 * q4 + j], b0, b1);
        }
      }
      const float by = q_scale * sk[nt / 2];
      sc[nt] = mul2(add2(make_float2(acc[0], acc[1]), make_float2(acc[2], acc[3])),
                    make_float2(by, by));
    }
    if (seen < TR) {
#pragma unroll
      for (int nt = 0; nt < TR / 8; ++nt) {
        if (nt * 8 + 2 * c >= seen) sc[nt].x = -INFINITY;
        if (nt * 8 + 2 * c + 1 >= seen) sc[nt].y = -INFINITY;
      }
      if constexpr (FMT == PL_KV8_E4M3) {
        // rows past the end weigh 0, but their bytes may be NaN codes
        for (int o = seen * HD + lane * 16; o < TR * HD; o += 512)
          asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(vt + o), "r"(0) : "memory");
        __syncwarp();
      }
    }
    // generic writes to the stage come before it is filled again
    if (appends || (FMT == PL_KV8_E4M3 && seen < TR)) fence_proxy_async_smem();
#pragma unroll
    for (int nt = 0; nt < TR / 8; ++nt) mt = max3(mt, sc[nt].x, sc[nt].y);
    mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 1));
    mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 2));
    const float m_new = fmaxf(st.m, mt);
    const float alpha = ex2(st.m - m_new);
    float top = sv[0];
#pragma unroll
    for (int b = 1; b < Sh::kBlocks; ++b)
      if (b * kBlock < seen) top = fmaxf(top, sv[b]);
    const float ref_new = fmaxf(ref, top);
    const float keep = alpha * (ref / ref_new), lift = kWeightScale / ref_new;
    ref = ref_new;
    st.m = m_new;
    // ---- the weights, as A fragments
    uint32_t pa[Sh::kBlocks][4];
    float2 sum = make_float2(0.f, 0.f);
    const float2 nm = make_float2(-m_new, -m_new);
#pragma unroll
    for (int b = 0; b < Sh::kBlocks; ++b) {
      const float by = b * kBlock < seen ? sv[b] * lift : 0.f;
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const float2 x = add2(sc[2 * b + hf], nm);
        const float2 p = make_float2(ex2(x.x), ex2(x.y));
        sum = add2(sum, p);
        const float2 w = mul2(p, make_float2(by, by));
        split_hi_lo(w.x, w.y, pa[b][2 * hf], pa[b][2 * hf + 1]);
      }
    }
    st.l = fmaf(st.l, alpha, sum.x + sum.y);
    // ---- O = O * keep + P V, 32 dims at a time
#pragma unroll
    for (int ch = 0; ch < HD / 16; ch += 2) {
      float ot[4][4];  // even and odd dims of chunk ch, then of ch + 1
#pragma unroll
      for (int b = 0; b < Sh::kBlocks; ++b) {
        uint32_t w[4];  // (rows 0-7, 8-15) of chunk ch, then of ch + 1
        ldmatrix_x4_trans(vt + tile_off<HD>(b * kBlock + ((lane >> 3) & 1) * 8 + (lane & 7),
                                            ch + (lane >> 4)),
                          w[0], w[1], w[2], w[3]);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t b0 = k & 1 ? codes_half2<FMT, 0x31>(w[k & 2]) : codes_half2<FMT, 0x20>(w[k & 2]);
          const uint32_t b1 =
              k & 1 ? codes_half2<FMT, 0x31>(w[(k & 2) + 1]) : codes_half2<FMT, 0x20>(w[(k & 2) + 1]);
          if (b == 0) mma_16816_zero(ot[k], pa[b], b0, b1);
          else mma_16816(ot[k], pa[b], b0, b1);
        }
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float* o = &st.o[4 * ch + 2 * k];
        const float2 t = fma2(make_float2(o[0], o[1]), make_float2(keep, keep),
                              add2(make_float2(ot[k][0], ot[k][1]), make_float2(ot[k][2], ot[k][3])));
        o[0] = t.x;
        o[1] = t.y;
      }
    }
    // ---- the stage is free: the next tile
    __syncwarp();
    if (issued < x1) {
      if (issued - t_base >= 32) place_tile(find_tile(issued));
      issue(issued);
      ++issued;
    }
    // ---- the segment's end
    if (x == run_last || x == x1 - 1) {
      st.l += __shfl_xor_sync(0xffffffffu, st.l, 1);
      st.l += __shfl_xor_sync(0xffffffffu, st.l, 2);
      const float back = ref * (1.f / kWeightScale);
#pragma unroll
      for (int d = 0; d < HD / 4; ++d) st.o[d] *= back;
      if (max(run_first, b0) < x0) {
        st.save(sm.part[warp], lane);  // the warp where the run starts takes it
      } else if (x == run_last && run_first >= b0) {
        const int tok = a.start ? a.start[i] : i;
        st.write(static_cast<T*>(a.out) + tok * a.out_stride + h * G * HD, lane, G);
      } else if (x != x1 - 1) {
        // the end of an earlier block's run, with more to do: left for later
        st.save(sm.part[warp], lane);
        if (lane == 0) {
          sm.ended[0] = run;
          sm.ended[1] = run_first;
          sm.ended[2] = run_last;
          sm.ended[3] = warp;
        }
      }
    }
  }
  // never leave with copies in flight
  for (int x = max(issued - NS, x0); x < issued; ++x)
    mbar_wait_drained(&sm.full[warp][(x - x0) % NS], ((x - x0) / NS) & 1);
  __syncthreads();

  auto write_run = [&](int r) {
    const int i = r / heads, h = r - i * heads, tok = a.start ? a.start[i] : i;
    st.write(static_cast<T*>(a.out) + tok * a.out_stride + h * G * HD, lane, G);
  };
  // The p-th block's partial of the run with first tile `first` in block f0.
  auto partial = [&](int f0, int p, int first) {
    const int slot = 2 * (f0 + p) + (first >= work.begin(f0 + p) ? 1 : 0);
    return da.part + static_cast<long long>(slot) * Sh::kPartFloats;
  };
  // `st` is this block's partial of a run over several blocks (kind 0: one
  // that started before the block, 1: in it).  The block that leaves the
  // last one merges them in the order of the blocks: a few at once here,
  // more of them with all warps below.
  auto publish = [&](int r, int first, int last, int kind) {
    st.save(da.part + static_cast<long long>(2 * blk + kind) * Sh::kPartFloats, lane);
    const int f0 = work.block_of(first), parts = work.block_of(last) - f0 + 1;
    __syncwarp();
    int done = 0;
    if (lane == 0) {
      done = arrive_acq_rel(&da.arrived[f0]) == parts - 1;
      if (done) {
        da.arrived[f0] = 0;
        if (parts > 4) sm.finish[kind] = r;
      }
    }
    done = __shfl_sync(0xffffffffu, done, 0);
    if (done && parts <= 4) {
      st.clear();
      for (int p = 0; p < parts; p += 2) {
        const float* p0 = partial(f0, p, first);
        st.fold_two(p0, p + 1 < parts ? partial(f0, p + 1, first) : p0, p + 1 < parts, lane);
      }
      write_run(r);
    }
  };
  // ---- runs that go on past this warp's slice (or came from another block):
  // the warp where the block's part of the run starts folds in the others'
  if (ok && x0 < x1 && max(run_first, b0) >= x0 && (run_last >= x1 || run_first < b0)) {
    const int end = min(run_last + 1, b1);
    for (int w = warp + 1; w < W; ++w) {
      const int w0 = b0 + w * span / W, w1 = b0 + (w + 1) * span / W;
      if (w0 < w1 && w0 < end) st.fold_from(sm.part[w], lane);
    }
    if (run_first >= b0 && run_last < b1) write_run(run);
    else publish(run, run_first, run_last, run_first >= b0 ? 1 : 0);
  }
  if (sm.ended[0] >= 0 && warp == (sm.ended[3] + W / 2) % W) {
    st.clear();
    st.fold_from(sm.part[sm.ended[3]], lane);
    publish(sm.ended[0], sm.ended[1], sm.ended[2], 0);
  }
  __syncthreads();
  // ---- runs of many blocks: all warps merge their partials together
#pragma unroll 1
  for (int f = 0; f < 2; ++f) {
    const int r = sm.finish[f];
    if (r < 0) continue;
    const int i = r / heads, h = r - i * heads;
    const int tiles = (sm.prefix[i + 1] - sm.prefix[i]) / heads;
    const int first = sm.prefix[i] + h * tiles, f0 = work.block_of(first);
    const int parts = work.block_of(first + tiles - 1) - f0 + 1;
    st.clear();
    for (int p = warp; p < parts; p += 2 * W) {
      const bool two = p + W < parts;
      const float* p0 = partial(f0, p, first);
      st.fold_two(p0, two ? partial(f0, p + W, first) : p0, two, lane);
    }
    st.save(sm.part[warp], lane);
    __syncthreads();
    if (warp == 0) {
      for (int w = 1; w < W; ++w) st.fold_from(sm.part[w], lane);
      write_run(r);
    }
    __syncthreads();
  }
}

}  // namespace pl
